"""The operators of the paged cache held in 4 bits against plain implementations in 64 bits.

Writes are held to the format's formula byte for byte (each of its operations is one IEEE rounding).
Attention is held, value by value, to what its roundings allow: with o the exact output and A = sum_t p_t
max_d |v_td|, the bf16 result is within 2^-9 |o| (its own rounding), P * scale in f16 and the code sums
within 2^-10 A; prefill's P and V in bf16 within 2^-8 A, and its K in bf16 moves a score by noise of deviation
scale 2^-9 sqrt(sum_d (q_d k_td)^2 / 3), of which six are allowed, taken at the worst key. One bit is allowed
on top of the f16 figure.
"""

import math

import pytest
import torch

from everserve_b200.ops import KernelOps, ref

pytestmark = pytest.mark.gpu

# query heads, kv heads, head dim, group, block size
LAYOUTS = [(32, 8, 128, 64, 16), (32, 8, 128, 128, 32), (64, 8, 128, 64, 32), (14, 2, 64, 64, 16), (4, 4, 64, 64, 32),
           (20, 2, 128, 64, 16), (16, 1, 64, 64, 16)]


@pytest.fixture(scope="module")
def kops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return KernelOps("cuda:0")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def filled(nb, hkv, d, group, bs, g):
    """A cache of quantised rows, K with an offset of its own in every channel."""
    cache = torch.zeros(ref.kv4_cache_shape(nb, hkv, bs, d, group), dtype=torch.uint8, device="cuda")
    parts = ref.kv4_parts(cache, d, bs)
    lean = 2 * torch.randn(hkv, 1, d, device="cuda", generator=g)
    for i, off in ((0, lean), (1, 0.0)):
        c, p = ref.kv4_quantize(torch.randn(nb, hkv, bs, d, device="cuda", generator=g) + off, d // group)
        parts[i].copy_(c)
        parts[2 + i].copy_(p.flatten(-2).contiguous().view(torch.uint8))
    return cache


def poison(cache, d, bs, blocks, start):
    """NaN pairs in the rows from `start` on of each of `blocks` (what a freed page may hold)."""
    parts = ref.kv4_parts(cache, d, bs)
    for blk, s in zip(blocks, start):
        for p in parts[2:]:
            p[blk, :, s:] = 255


def batch(lens, rows, hq, hkv, d, group, bs, seed, extra_blocks=3):
    """q, cache, tables, ctx_lens, last_rows of sequences with those context lengths and new rows; slots
    past a history's end hold NaN."""
    g = gen(seed)
    held = [-(-n // bs) for n in lens]
    nb = sum(held) + extra_blocks
    cache = filled(nb, hkv, d, group, bs, g)
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seed))
    tables = torch.zeros(len(lens), max(1, max(held)), dtype=torch.int32)
    at = 0
    for i, h in enumerate(held):
        tables[i, :h] = perm[at : at + h].int()
        at += h
    poison(cache, d, bs, perm[at:].tolist(), [0] * extra_blocks)
    poison(cache, d, bs, [int(tables[i, h - 1]) for i, h in enumerate(held) if h],
           [n - (h - 1) * bs for n, h in zip(lens, held) if h])
    q = torch.randn(sum(rows), hq, d, device="cuda", generator=g).bfloat16()
    last = torch.tensor(rows).cumsum(0) - 1
    return q, cache, tables.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), last.cuda()


def oracle(q, cache, tables, lens, last, scale, bs):
    """(output, A) in 64 bits; rows without a visible key are zero."""
    T, hq, d = q.shape
    hkv = cache.shape[1]
    vals = ref.kv4_cache_values(cache, d, bs).double()
    out = torch.zeros(T, hq, d, dtype=torch.float64, device="cuda")
    mag = torch.zeros(T, hq, 1, dtype=torch.float64, device="cuda")
    r0 = 0
    for s, (r1, n) in enumerate(zip((last + 1).tolist(), lens.tolist())):
        if n:
            blk = tables[s, : -(-n // bs)].long()
            k, v = (vals[blk, i].transpose(1, 2).reshape(-1, hkv, d)[:n].repeat_interleave(hq // hkv, 1) for i in (0, 1))
            a = torch.einsum("thd,nhd->htn", q[r0:r1].double(), k) * scale
            pos = torch.arange(n - (r1 - r0), n, device="cuda")
            a = a.masked_fill((torch.arange(n, device="cuda")[None] > pos[:, None])[None], -math.inf)
            p = torch.softmax(a, -1)
            o, m = torch.einsum("htn,nhd->thd", p, v), torch.einsum("htn,nh->th", p, v.abs().amax(-1))[..., None]
            seen = (pos >= 0)[:, None, None]
            out[r0:r1], mag[r0:r1] = torch.where(seen, o, 0), torch.where(seen, m, 0)
        r0 = r1
    return out, mag


def held_to(got, want, mag, of_mag):
    err = (got.double() - want).abs()
    tol = 2.0**-8 * want.abs() + of_mag * mag + 1e-30
    assert bool(torch.isfinite(got).all())
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} of the bound"


DECODE_MAG = 2.0**-9


@pytest.mark.parametrize("hq,hkv,d,group,bs", LAYOUTS)
def test_decode(kops, hq, hkv, d, group, bs):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 255, 256, 257, 300, 512, 513, 1000, 2049, 4097]
    q, cache, tables, ctx, last = batch(lens, [1] * len(lens), hq, hkv, d, group, bs, 7)
    scale = d**-0.5
    out = kops.decode_attention_kv4(q, cache, tables, ctx, scale, bs)
    want, mag = oracle(q, cache, tables, ctx, last, scale, bs)
    assert kops.check_status() == 0
    held_to(out, want, mag, DECODE_MAG)
    assert not bool(out[0].any())  # an empty history
    # the same bits again, alone in its batch, and whatever the longest length allowed
    assert torch.equal(out, kops.decode_attention_kv4(q, cache, tables, ctx, scale, bs))
    for i in (1, 13, 19):
        one = kops.decode_attention_kv4(q[i : i + 1], cache, tables[i : i + 1], ctx[i : i + 1], scale, bs, 8192)
        assert torch.equal(out[i], one[0])


def test_decode_extremes(kops):
    """Scores far apart (one key takes all, in the first, a middle or the last run), scales that grow
    and shrink by 2^30 along the history, zero scales, huge and tiny queries."""
    hq, hkv, d, group, bs = 8, 2, 128, 64, 16
    lens = [1200, 700, 530, 90, 1300]
    q, cache, tables, ctx, last = batch(lens, [1] * len(lens), hq, hkv, d, group, bs, 11)
    parts = ref.kv4_parts(cache, d, bs)
    kp, vp = (p.view(torch.bfloat16) for p in parts[2:])  # [nb, hkv, bs, 2 * groups]
    for j, at in ((0, 3), (0, 700), (1, 699)):
        kp[tables[j, at // bs].long(), :, at % bs] *= 30
    vp[tables[2].long()[:: 3]] *= 2.0**15
    vp[tables[2].long()[1::3]] *= 2.0**-15
    vp[tables[3].long()[:6], :, :, 0::2] = 0  # constant groups
    kp[tables[3].long()[:6], :, :, 0::2] = 0
    q[4] *= 2.0**20
    q[3] *= 2.0**-20
    q[1, 0] = 0
    scale = d**-0.5
    out = kops.decode_attention_kv4(q, cache, tables, ctx, scale, bs)
    want, mag = oracle(q, cache, tables, ctx, last, scale, bs)
    held_to(out, want, mag, DECODE_MAG)


@pytest.mark.parametrize("group", [64, 128])
def test_decode_averages_of_long_histories(kops, group):
    """What 50K keys of like weight average to is a hundredth of their codes' sum, so nothing may lean one
    way. Over all values: bf16's rounding, 0.0017 of the norm, and the noise of P * scale in f16, 0.0005
    (2^-12 / sqrt 3 of scale * code, 3.4 times the values' own deviation), at half as much again."""
    hq, hkv, d, bs = 32, 8, 128, 16
    q, cache, tables, ctx, last = batch([50001, 49000], [1, 1], hq, hkv, d, group, bs, 14)
    out = kops.decode_attention_kv4(q, cache, tables, ctx, d**-0.5, bs)
    want, _ = oracle(q, cache, tables, ctx, last, d**-0.5, bs)
    assert float((out.double() - want).norm() / want.norm()) < 1.5 * (0.0017**2 + 0.0005**2) ** 0.5


def test_decode_nan_stays_in_its_sequence(kops):
    hq, hkv, d, group, bs = 8, 2, 64, 64, 16
    q, cache, tables, ctx, last = batch([100, 100, 100], [1] * 3, hq, hkv, d, group, bs, 12)
    want, mag = oracle(q, cache, tables, ctx, last, 0.125, bs)
    poison(cache, d, bs, [int(tables[1, 2])], [5])
    out = kops.decode_attention_kv4(q, cache, tables, ctx, 0.125, bs)
    assert bool(out[1].isnan().all())
    for i in (0, 2):
        held_to(out[i], want[i], mag[i], DECODE_MAG)


def test_strides_and_far_pages(kops):
    """q rows out of a wider tensor, a layer's cache out of an interleaved one, pages beyond 4 GiB."""
    hq, hkv, d, group, bs = 32, 8, 128, 64, 16
    lens = [77, 300]
    q, cache, tables, ctx, last = batch(lens, [1, 1], hq, hkv, d, group, bs, 13)
    wide = torch.zeros(2, hq * d + 64, dtype=torch.bfloat16, device="cuda")
    wide[:, : hq * d] = q.flatten(1)
    nb, far = cache.shape[0], (5 << 30) // (2 * cache[0].numel())
    both = torch.zeros(far + nb, 2, *cache.shape[1:], dtype=torch.uint8, device="cuda")
    both[far:, 1] = cache
    layer = both[:, 1]
    tables += far
    out = kops.decode_attention_kv4(wide[:, : hq * d].unflatten(1, (hq, d)), layer, tables, ctx, d**-0.5, bs)
    want, mag = oracle(q, cache, tables - far, ctx, last, d**-0.5, bs)
    held_to(out, want, mag, DECODE_MAG)
    slots = tables[1, :2].long() * bs + torch.tensor([3, 15], device="cuda")
    k, v = kops.kv4_read(layer, slots, d, bs)
    wk, wv = ref.kv4_read(cache, slots - far * bs, d, bs)
    assert torch.equal(k, wk.bfloat16()) and torch.equal(v, wv.bfloat16())
    pairs = torch.tensor([[far, far + nb - 1]], device="cuda")
    was = both[:, 0].sum(dtype=torch.int64)
    kops.copy_pages([layer], pairs)
    assert torch.equal(layer[far + nb - 1], layer[far]) and both[:, 0].sum(dtype=torch.int64) == was


@pytest.mark.parametrize("hq,hkv,d,group,bs", LAYOUTS)
@pytest.mark.parametrize("T,bias", [(1, False), (37, True), (1000, False)])
def test_write_and_read(kops, hq, hkv, d, group, bs, T, bias):
    g = gen(T + hq)
    width = (hq + 2 * hkv) * d
    wide = torch.randn(T, width + 8, device="cuda", generator=g).bfloat16()
    qkv = wide[:, :width]  # rows apart
    qkv[T // 2, hq * d : (hq + 1) * d] = 3.0  # a constant row before the rotation
    qkv[T // 2, -d:] = 1.25  # and one of V: scale 0
    b = torch.randn(width, device="cuda", generator=g).bfloat16() if bias else None
    cs = ref.cos_sin_table(d, 4096, 5e5).cuda()
    pos = torch.randint(0, 4096, (T,), device="cuda", generator=g)
    nb = T // bs + 3
    slots = torch.randperm(nb * bs, device="cuda", generator=g)[:T]
    if T > 1:
        slots[3] = -1
    cache = torch.full(ref.kv4_cache_shape(nb, hkv, bs, d, group), 0xA5, dtype=torch.uint8, device="cuda")
    want = cache.clone()
    q = kops.rope_kv4_write(qkv, b, pos, cs, slots, cache, hq, hkv, bs)
    wq = ref.rope_kv4_write(qkv, b, pos, cs, slots, want, hq, hkv, bs)
    assert kops.check_status() == 0
    assert torch.equal(q, wq)
    assert torch.equal(cache, want)  # the other slots' bytes among them
    k, v = kops.kv4_read(cache, slots, d, bs)
    wk, wv = ref.kv4_read(want, slots, d, bs)
    assert torch.equal(k, wk.bfloat16()) and torch.equal(v, wv.bfloat16())
    # what is held is within half a step of what was written, but for the bf16 scale and zero
    x = (qkv.float() + (b.float() if bias else 0)).view(T, hq + 2 * hkv, d)[:, hq + hkv :].double()
    grp = x.unflatten(-1, (d // group, group))
    step = (grp.amax(-1) - grp.amin(-1)) / 15
    tol = 0.5 * step + 15 * step * 2.0**-9 + grp.abs().amax(-1) * 2.0**-8
    keep = slots >= 0
    off = (v.double().unflatten(-1, (d // group, group)) - grp).abs().amax(-1)
    assert bool((off <= tol)[keep].all()) and not bool(v[~keep].any())


def test_write_not_finite(kops):
    """A value that is not finite makes its group read as NaN, and no other."""
    hq, hkv, d, bs = 2, 2, 128, 16
    qkv = torch.randn(3, (hq + 2 * hkv) * d, device="cuda").bfloat16()
    qkv[0, -1], qkv[1, -d], qkv[2, -d - 1] = math.inf, math.nan, -math.inf
    cs = ref.cos_sin_table(d, 64, 1e4).cuda()
    cache = torch.zeros(ref.kv4_cache_shape(1, hkv, bs, d), dtype=torch.uint8, device="cuda")
    slots = torch.arange(3, device="cuda")
    kops.rope_kv4_write(qkv, None, slots, cs, slots, cache, hq, hkv, bs)
    k, v = kops.kv4_read(cache, slots, d, bs)
    bad = torch.zeros(3, hkv, 2, 64, dtype=torch.bool, device="cuda")
    bad[0, 1, 1] = bad[1, 1, 0] = bad[2, 0, 1] = True
    assert torch.equal(v.isnan(), bad.view(3, hkv, d)) and not bool(k.isnan().any())


def test_out_of_range_is_reported(kops):
    hq, hkv, d, bs = 4, 2, 64, 16
    cache = torch.zeros(ref.kv4_cache_shape(2, hkv, bs, d), dtype=torch.uint8, device="cuda")
    cs = ref.cos_sin_table(d, 64, 1e4).cuda()
    one = torch.zeros(1, dtype=torch.int64, device="cuda")
    qkv = torch.ones(1, (hq + 2 * hkv) * d, device="cuda").bfloat16()
    assert kops.check_status() == 0
    kops.rope_kv4_write(qkv, None, one, cs, one + 32, cache, hq, hkv, bs)
    assert kops.check_status() == 3 and not bool(cache.any())
    kops.rope_kv4_write(qkv, None, one + 64, cs, one - 1, cache, hq, hkv, bs)
    assert kops.check_status() == 3
    kops.kv4_read(cache, one + 40, d, bs)
    assert kops.check_status() == 3
    kops.decode_attention_kv4(torch.ones(1, hq, d, device="cuda").bfloat16(), cache, (one + 2).int()[None], (one + 5).int(),
                              0.1, bs)
    assert kops.check_status() == 3
    kops.copy_pages([cache], torch.tensor([[0, 2]], device="cuda"))
    assert kops.check_status() == 3


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("layers,n,hkv,d,bs", [(1, 1, 2, 64, 16), (24, 7, 8, 128, 32), (257, 3, 1, 64, 16), (2, 301, 8, 128, 16)])
def test_copy_pages(kops, kind, layers, n, hkv, d, bs):
    g = gen(n)
    nb = 2 * n + 2
    if kind == "bf16":
        caches = [torch.randn(nb, 2, hkv, bs, d, device="cuda", generator=g).bfloat16() for _ in range(layers)]
    else:
        shape = ref.kv4_cache_shape(nb, hkv, bs, d)
        caches = [torch.randint(0, 256, shape, device="cuda", generator=g, dtype=torch.uint8) for _ in range(layers)]
    order = torch.randperm(nb, device="cuda", generator=g)
    pairs = torch.stack((order[:n], order[n : 2 * n]), 1).contiguous()
    if n > 1:
        pairs[1] = -1
    want = [c.clone() for c in caches]
    ref.copy_pages(want, pairs)
    kops.copy_pages(caches, pairs)
    assert kops.check_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(caches, want))
    kops.copy_pages(caches, pairs[:0])


def prefill_mag(q, cache, tables, lens, last, scale, bs):
    """2^-8 and six deviations of a score's noise, per row and head."""
    hq, d = q.shape[1:]
    vals = ref.kv4_cache_values(cache, d, bs).double()
    out = torch.zeros(q.shape[0], hq, 1, dtype=torch.float64, device="cuda")
    r0 = 0
    for s, (r1, n) in enumerate(zip((last + 1).tolist(), lens.tolist())):
        if n:
            k = vals[tables[s, : -(-n // bs)].long(), 0].transpose(1, 2).reshape(-1, cache.shape[1], d)[:n]
            sq = torch.einsum("thd,nhd->thn", q[r0:r1].double() ** 2, k.repeat_interleave(hq // cache.shape[1], 1) ** 2)
            out[r0:r1] = sq.amax(-1, keepdim=True)
        r0 = r1
    return 2.0**-8 + 6 * 2.0**-9 * scale * (out / 3).sqrt()


@pytest.mark.parametrize("hq,hkv,d,group,bs", LAYOUTS)
def test_prefill(kops, hq, hkv, d, group, bs):
    """Rows from one to several tiles, histories from none to long (cut along the keys), ends inside tiles
    and blocks, a sequence without keys, one with more rows than keys."""
    rows = [1, 2, 31, 64, 127, 128, 129, 300, 1, 5, 33, 70, 1, 9, 600]
    past = [0, 0, 0, 0, 1, 0, 15, 0, 700, 1027, 2300, 5000, -1, -4, 200]
    lens = [r + p for r, p in zip(rows, past)]
    q, cache, tables, ctx, last = batch(lens, rows, hq, hkv, d, group, bs, 31)
    scale = d**-0.5
    out = kops.prefill_attention_kv4(q, cache, tables, ctx, last, scale, bs)
    assert kops.check_status() == 0
    want, mag = oracle(q, cache, tables, ctx, last, scale, bs)
    held_to(out, want, mag, prefill_mag(q, cache, tables, ctx, last, scale, bs))
    at = sum(rows[:13])
    assert not bool(out[at : at + 4].any()) and not bool(out[at - 1].any())  # no visible key
    assert torch.equal(out, kops.prefill_attention_kv4(q, cache, tables, ctx, last, scale, bs))
    # a sequence alone gives the same bits
    for s in (4, 7, 11):
        r0 = sum(rows[:s])
        one = kops.prefill_attention_kv4(q[r0 : r0 + rows[s]], cache, tables[s : s + 1], ctx[s : s + 1],
                                         last[s : s + 1] - r0, scale, bs)
        assert torch.equal(one, out[r0 : r0 + rows[s]])


def test_prefill_many_sequences_and_long(kops):
    """More sequences than a warp scans at once, and a prompt of several thousand rows."""
    hq, hkv, d, group, bs = 8, 2, 128, 64, 16
    rows = [1 + i % 5 for i in range(70)]
    lens = [r + 7 * i for i, r in enumerate(rows)]
    q, cache, tables, ctx, last = batch(lens, rows, hq, hkv, d, group, bs, 32)
    out = kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs)
    want, mag = oracle(q, cache, tables, ctx, last, 0.1, bs)
    held_to(out, want, mag, prefill_mag(q, cache, tables, ctx, last, 0.1, bs))
    q, cache, tables, ctx, last = batch([5003], [5003], hq, hkv, d, group, bs, 33)
    out = kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs)
    want, mag = oracle(q, cache, tables, ctx, last, 0.1, bs)
    held_to(out, want, mag, prefill_mag(q, cache, tables, ctx, last, 0.1, bs))
    assert kops.check_status() == 0


def test_prefill_extremes(kops):
    """Maxima that move late and far (the output is rescaled), and scores equal to the last bit."""
    hq, hkv, d, group, bs = 4, 1, 128, 128, 16
    q, cache, tables, ctx, last = batch([1500, 400], [300, 400], hq, hkv, d, group, bs, 34)
    kp = ref.kv4_parts(cache, d, bs)[2].view(torch.bfloat16)
    for key in (200, 900, 1290):
        kp[tables[0, key // bs].long(), :, key % bs] *= 12
    q[300:] = 0  # every key alike
    out = kops.prefill_attention_kv4(q, cache, tables, ctx, last, d**-0.5, bs)
    want, mag = oracle(q, cache, tables, ctx, last, d**-0.5, bs)
    held_to(out, want, mag, prefill_mag(q, cache, tables, ctx, last, d**-0.5, bs))
    assert kops.check_status() == 0


def test_other_stream_and_graph(kops):
    """A call on a side stream, and a captured one replayed on new lengths and contents."""
    hq, hkv, d, group, bs = 32, 8, 128, 64, 16
    lens = [1000, 20, 513]
    q, cache, tables, ctx, last = batch(lens, [1] * 3, hq, hkv, d, group, bs, 21)
    main = kops.decode_attention_kv4(q, cache, tables, ctx, 0.1, bs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = [kops.decode_attention_kv4(q, cache, tables, ctx, 0.1, bs) for _ in range(3)]
    here = [kops.decode_attention_kv4(q * 2, cache, tables, ctx, 0.05, bs) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(main, x) for x in side + here)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kops.decode_attention_kv4(q, cache, tables, ctx, 0.1, bs)
    q.copy_(q.flip(0))
    ctx.copy_(torch.tensor([257, 0, 512], dtype=torch.int32))
    g.replay()
    assert torch.equal(out, kops.decode_attention_kv4(q, cache, tables, ctx, 0.1, bs))
    want, mag = oracle(q, cache, tables, ctx, last, 0.1, bs)
    held_to(out, want, mag, DECODE_MAG)


def test_refusals(kops):
    hq, hkv, d, bs = 4, 2, 64, 16
    dev = "cuda"
    cache = torch.zeros(ref.kv4_cache_shape(3, hkv, bs, d), dtype=torch.uint8, device=dev)
    q = torch.zeros(1, hq, d, dtype=torch.bfloat16, device=dev)
    bt, ctx = torch.zeros(1, 2, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)

    def decode(q=q, cache=cache, bt=bt, ctx=ctx, bs=bs):
        return kops.decode_attention_kv4(q, cache, bt, ctx, 0.1, bs)

    decode()
    for bad in (dict(q=q.float()), dict(q=q[..., :32]), dict(q=q[:, :3]), dict(cache=cache.cpu()), dict(cache=cache[..., :-8]),
                dict(cache=cache.float()), dict(bs=32), dict(bs=8), dict(bt=bt.long()), dict(ctx=ctx.long()),
                dict(bt=bt.cpu()), dict(bt=bt[:0]), dict(cache=cache[:, :, 16:])):
        with pytest.raises(RuntimeError):
            decode(**bad)
    cs = ref.cos_sin_table(d, 64, 1e4).cuda()
    i = torch.zeros(1, dtype=torch.int64, device=dev)
    qkv = torch.zeros(1, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device=dev)
    for bad in (dict(qkv=qkv[:, :-d]), dict(pos=i.int()), dict(slots=i[:0]), dict(hkv=1), dict(cs=cs.cpu()),
                dict(cs=cs.double()), dict(bias=qkv[0, :d])):
        a = dict(qkv=qkv, bias=None, pos=i, cs=cs, slots=i, hkv=hkv)
        a.update(bad)
        with pytest.raises(RuntimeError):
            kops.rope_kv4_write(a["qkv"], a["bias"], a["pos"], a["cs"], a["slots"], cache, hq, a["hkv"], bs)
    with pytest.raises(RuntimeError):
        kops.kv4_read(cache, i.int(), d, bs)
    for bad in (dict(last=i.int()), dict(last=torch.cat([i, i])), dict(scale=0.0), dict(q=q.float())):
        a = dict(q=q, last=i, scale=0.1)
        a.update(bad)
        with pytest.raises(RuntimeError):
            kops.prefill_attention_kv4(a["q"], cache, bt, ctx, a["last"], a["scale"], bs)
    for caches, pairs in (([cache, cache[:2]], torch.zeros(1, 2, dtype=torch.int64, device=dev)),
                          ([cache[:, :, 16:32]], torch.zeros(1, 2, dtype=torch.int64, device=dev)),
                          ([cache], torch.zeros(1, 2, dtype=torch.int32, device=dev)),
                          ([cache], torch.zeros(2, dtype=torch.int64, device=dev))):
        with pytest.raises(RuntimeError):
            kops.copy_pages(caches, pairs)

"""Prefill attention over the paged cache held in 4 bits, where rows and keys are out of the ordinary.

Values are held to what the kernel's f16 operands allow. With o the exact output, A = sum_t p_t max_d |v_td| and
u = 2^-11 the rounding of f16: the bf16 result is within 2^-8 |o|; P and V are each rounded once, 2 u A; a key's
value is off by a uniform error of at most u |k|, which moves its score by noise of deviation
scale u sqrt(sum_d (q_d k_td)^2 / 3), of which six are allowed for the worst key, and a score's shift moves the output
by at most itself times (A + |o|).
"""

import math

import pytest
import torch

from everserve_b200.ops import KernelOps, ref
from test_kv4_gpu import batch, oracle

pytestmark = pytest.mark.gpu

# query heads, kv heads, head dim, group, block size
LAYOUTS = [(8, 2, 128, 64, 16), (8, 2, 128, 128, 32), (14, 2, 64, 64, 16)]


@pytest.fixture(scope="module")
def kops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return KernelOps("cuda:0")


def bound(q, cache, tables, lens, last, scale, bs, want, mag):
    """The tolerance above, value by value."""
    T, hq, d = q.shape
    vals = ref.kv4_cache_values(cache, d, bs).double()
    worst = torch.zeros(T, hq, 1, dtype=torch.float64, device="cuda")
    r0 = 0
    for s, (r1, n) in enumerate(zip((last + 1).tolist(), lens.tolist())):
        if n:
            k = vals[tables[s, : -(-n // bs)].long(), 0].transpose(1, 2).reshape(-1, cache.shape[1], d)[:n]
            sq = torch.einsum("thd,nhd->thn", q[r0:r1].double() ** 2, k.repeat_interleave(hq // cache.shape[1], 1) ** 2)
            worst[r0:r1] = sq.amax(-1, keepdim=True)
        r0 = r1
    shift = 6 * 2.0**-11 * scale * (worst / 3).sqrt()
    return 2.0**-8 * want.abs() + 2 * 2.0**-11 * mag + shift * (mag + want.abs()) + 1e-30


def held_to(got, want, tol):
    err = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} of the bound"


def pairs_of(cache, d, bs):
    """K's and V's (scale, zero) pairs, bf16 [blocks, kv heads, bs, 2 * groups]."""
    return [p.view(torch.bfloat16) for p in ref.kv4_parts(cache, d, bs)[2:]]


@pytest.mark.parametrize("hq,hkv,d,group,bs", LAYOUTS)
def test_not_finite_reaches_the_rows_that_see_it(kops, hq, hkv, d, group, bs):
    """Groups holding a value that is not finite (as the write leaves them: NaN scale, a zero that may be
    -infinity) in keys that some rows of their tile see and others do not: a key's K makes the rows that see
    it NaN, its V the group's channels of those rows, and no other row moves. Whole and cut histories."""
    rows, lens = [300, 40], [300, 2040]
    q, cache, tables, ctx, last = batch(lens, rows, hq, hkv, d, group, bs, 41)
    scale, ng, G = d**-0.5, d // group, hq // hkv
    want, mag = oracle(q, cache, tables, ctx, last, scale, bs)
    tol = bound(q, cache, tables, ctx, last, scale, bs, want, mag)
    kp, vp = pairs_of(cache, d, bs)
    bad = torch.zeros(sum(rows), hkv, G, ng, group, dtype=torch.bool, device="cuda")

    def plant(pairs, seq, key, head, grp, pair):
        pairs[tables[seq, key // bs].long(), head, key % bs, 2 * grp : 2 * grp + 2] = torch.tensor(pair, device="cuda").bfloat16()
        first = sum(rows[:seq])
        seen = first + max(0, key - (lens[seq] - rows[seq]))
        sel = bad[seen : first + rows[seq], head]
        (sel if pairs is kp else sel[:, :, grp])[...] = True

    plant(vp, 0, 200, 0, 0, (math.nan, 0.5))
    plant(vp, 0, 230, 0, ng - 1, (math.nan, -math.inf))
    plant(kp, 0, 250, 0, 0, (math.nan, -math.inf))
    plant(vp, 0, 290, 1, 0, (math.nan, math.nan))
    plant(vp, 1, 2010, 1, ng - 1, (math.nan, -math.inf))
    plant(kp, 1, 2030, 0, 0, (math.nan, math.nan))
    out = kops.prefill_attention_kv4(q, cache, tables, ctx, last, scale, bs)
    bad = bad.view(sum(rows), hq, d)
    assert torch.equal(out.isnan(), bad)
    held_to(out.masked_fill(bad, 0), want.masked_fill(bad, 0), tol)
    assert kops.check_status() == 0
    # and a tile of the next call starts clean
    for p in (kp, vp):
        p.nan_to_num_(1.0, 1.0, 1.0)
    assert bool(torch.isfinite(kops.prefill_attention_kv4(q, cache, tables, ctx, last, scale, bs)).all())


def test_rows_of_no_sequence_are_zero(kops):
    """Rows past the last sequence's, whatever the output's memory held."""
    hq, hkv, d, group, bs = 8, 2, 128, 64, 16
    q, cache, tables, ctx, last = batch([200, 5020], [100, 20], hq, hkv, d, group, bs, 42)
    want = kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs)
    more = torch.cat([q, torch.ones(77, hq, d, device="cuda").bfloat16()])
    for seqs, rows in ((2, 120), (1, 100), (0, 0)):
        torch.full((64 << 20,), math.nan, device="cuda")  # what the allocator hands out next
        out = kops.prefill_attention_kv4(more, cache, tables, ctx, last[:seqs], 0.1, bs)
        assert torch.equal(out[:rows], want[:rows]) and not bool(out[rows:].any())
    assert kops.check_status() == 0


def test_visible_scores_of_minus_infinity(kops):
    """A query whose scores all come to -infinity has NaN as its softmax, not the zeros of a row without keys."""
    hq, hkv, d, group, bs = 2, 1, 64, 64, 16
    q, cache, tables, ctx, last = batch([1, 3000], [1, 3], hq, hkv, d, group, bs, 43)
    kp, _ = pairs_of(cache, d, bs)
    kp[..., 1] = -100.0  # every channel of every key below zero
    kp[..., 0] = 1.0
    q = q.abs()
    q[:, 0, 5] = math.inf
    out = kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs)
    assert bool(out[:, 0].isnan().all()) and bool(torch.isfinite(out[:, 1]).all())
    assert kops.check_status() == 0


def test_workspace_is_what_the_step_needs(kops):
    """A prompt that is not cut beside one row over a long history: 65 MB of output, and no workspace to speak of
    when the lengths are given; without them no more than two sequences can take. Results do not move."""
    hq, hkv, d, group, bs = 32, 8, 128, 64, 16
    rows, lens = [8000, 1], [8000, 8001]
    q, cache, tables, ctx, last = batch(lens, rows, hq, hkv, d, group, bs, 44)
    outs = []
    for lengths, most in ((None, 200 << 20), (list(zip(rows, lens)), 2 << 20)):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        kw = {} if lengths is None else dict(lengths=lengths)
        outs.append(kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs, **kw))
        assert torch.cuda.max_memory_allocated() - before <= q.numel() * 2 + most
    assert torch.equal(*outs)
    one = kops.prefill_attention_kv4(q[8000:], cache, tables[1:], ctx[1:], last[1:] - 8000, 0.1, bs)
    assert torch.equal(one, outs[0][8000:])
    # 16 sequences of 128 rows on 16K keys: each at most 51 MB of parts
    q, cache, tables, ctx, last = batch([16400 + i for i in range(16)], [128] * 16, hq, hkv, d, group, bs, 45)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    full = kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs)
    assert torch.cuda.max_memory_allocated() - before <= 16 * (51 << 20)
    del full
    assert kops.check_status() == 0


def test_lengths_that_fall_short_are_safe(kops):
    """Lengths below the step's leave sequences uncut, with the same values within the roundings."""
    hq, hkv, d, group, bs = 8, 2, 128, 64, 16
    rows, lens = [5, 40, 1, 30], [3000, 2500, 4000, 200]
    q, cache, tables, ctx, last = batch(lens, rows, hq, hkv, d, group, bs, 46)
    want, mag = oracle(q, cache, tables, ctx, last, 0.1, bs)
    tol = bound(q, cache, tables, ctx, last, 0.1, bs, want, mag)
    full = kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs)
    held_to(full, want, tol)
    assert torch.equal(full, kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs, lengths=list(zip(rows, lens))))
    for lengths in ([(0, 0)] * 4, [(5, 3000), (0, 0), (0, 0), (0, 0)], [(1, 2048)] * 4):
        held_to(kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs, lengths=lengths), want, tol)
    for bad in ([(5, 3000)], []):
        with pytest.raises(RuntimeError):
            kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs, lengths=bad)
    assert kops.check_status() == 0


# Over many values of long histories, where an output is a small part of A: bf16's rounding has 0.0017 of the norm. P's
# and V's roundings are noise of u / sqrt 3 times 0.75 (a value's place in its binade) of what they round, 2.1e-4 each. A
# key's moves its score by 2.1e-4 sqrt(d) scale sqrt(5) = 4.7e-4 (these keys have a second moment of 5), and the output by as
# much of itself. Half as much again is allowed.
AVERAGE = 1.5 * (0.0017**2 + 2 * 0.00021**2 + 0.00047**2) ** 0.5


@pytest.mark.parametrize("hq,hkv,d,group,bs", [(32, 8, 128, 64, 16), (32, 8, 128, 128, 32), (14, 2, 64, 64, 16)])
def test_averages_of_long_histories(kops, hq, hkv, d, group, bs):
    """Histories cut along their keys (40 rows on 40K) and whole (1100 rows on 4K)."""
    rows, lens = [40, 1100], [40040, 5100]
    q, cache, tables, ctx, last = batch(lens, rows, hq, hkv, d, group, bs, 51)
    out = kops.prefill_attention_kv4(q, cache, tables, ctx, last, d**-0.5, bs)
    want, _ = oracle(q, cache, tables, ctx, last, d**-0.5, bs)
    for part in (slice(0, 40), slice(40, None)):
        assert float((out[part].double() - want[part]).norm() / want[part].norm()) < AVERAGE
    assert kops.check_status() == 0


@pytest.mark.parametrize("hq,hkv,d,group,bs", LAYOUTS)
def test_sizes_far_apart(kops, hq, hkv, d, group, bs):
    """Pages whose values are 2^15 and 2^-15 of the others', within tiles, between them and between the parts of a cut
    history; groups of equal values; queries of 2^30 on keys of 2^-30 and the other way round; rows of zeros.
    Values far below the largest one met so far may lose the bits under 2^-33 of it."""
    rows, lens = [300, 20, 150, 150, 9], [300, 5000, 400, 400, 3100]
    q, cache, tables, ctx, last = batch(lens, rows, hq, hkv, d, group, bs, 52)
    kp, vp = pairs_of(cache, d, bs)
    page = lambda s, at: tables[s, at].long()  # noqa: E731
    per = 128 // bs  # pages of a key tile
    used = [tables[s, : -(-n // bs)].long() for s, n in enumerate(lens)]
    vp[used[0][1::3]] *= 2.0**15  # within every tile
    vp[used[0][2::3]] *= 2.0**-15
    for tile in range(0, len(used[1]) // per, 3):  # between tiles, and so between the parts
        vp[used[1][tile * per : (tile + 1) * per]] *= 2.0**15
        vp[used[1][(tile + 1) * per : (tile + 2) * per]] *= 2.0**-15
    vp[used[4][: 8 * per]] *= 2.0**-15  # from small to large
    vp[used[4][16 * per :]] *= 2.0**15
    first = torch.tensor(rows).cumsum(0) - torch.tensor(rows)
    kp[used[2]] *= 2.0**-30
    q[first[2] : first[2] + 150] *= 2.0**30
    kp[used[3]] *= 2.0**30
    q[first[3] : first[3] + 150] *= 2.0**-30
    vp[page(3, 2), :, :, 0::2] = 0  # scale 0: equal values
    kp[page(3, 3), :, :, 0::2] = 0
    q[5] = 0
    q[first[1] + 3, 0] = 0
    scale = d**-0.5
    out = kops.prefill_attention_kv4(q, cache, tables, ctx, last, scale, bs)
    want, mag = oracle(q, cache, tables, ctx, last, scale, bs)
    tol = bound(q, cache, tables, ctx, last, scale, bs, want, mag)
    vals = ref.kv4_cache_values(cache, d, bs)
    for s in range(len(rows)):
        top = torch.nan_to_num(vals[used[s], 1]).abs().amax()
        tol[first[s] : first[s] + rows[s]] += lens[s] * 2.0**-33 * float(top)
    held_to(out, want, tol)
    assert kops.check_status() == 0


def test_strides_and_far_pages(kops):
    """q rows out of a wider tensor, a layer's cache out of an interleaved one, pages beyond 4 GiB."""
    hq, hkv, d, group, bs = 32, 8, 128, 64, 16
    rows, lens = [70, 5], [200, 2500]
    q, cache, tables, ctx, last = batch(lens, rows, hq, hkv, d, group, bs, 53)
    want = kops.prefill_attention_kv4(q, cache, tables, ctx, last, 0.1, bs)
    wide = torch.full((75, hq * d + 64), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, : hq * d] = q.flatten(1)
    nb, far = cache.shape[0], (5 << 30) // (2 * cache[0].numel())
    both = torch.zeros(far + nb, 2, *cache.shape[1:], dtype=torch.uint8, device="cuda")
    both[far:, 1] = cache
    tables += far
    out = kops.prefill_attention_kv4(wide[:, : hq * d].unflatten(1, (hq, d)), both[:, 1], tables, ctx, last, 0.1, bs)
    assert torch.equal(out, want) and kops.check_status() == 0


def test_other_stream(kops):
    """Calls on two streams at once do not meet: their items are handed out and their parts kept apart."""
    hq, hkv, d, group, bs = 32, 8, 128, 64, 16
    q, cache, tables, ctx, last = batch([900, 6000, 300], [500, 30, 1], hq, hkv, d, group, bs, 54)
    args = (cache, tables, ctx, last)
    want = kops.prefill_attention_kv4(q, *args, 0.1, bs), kops.prefill_attention_kv4(q, *args, 0.3, bs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = [kops.prefill_attention_kv4(q, *args, 0.3, bs) for _ in range(4)]
    here = [kops.prefill_attention_kv4(q, *args, 0.1, bs) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[0]) for x in here) and all(torch.equal(x, want[1]) for x in side)
    assert kops.check_status() == 0


def test_a_bad_table_entry_is_reported(kops):
    """Block 0 is read in its place; rows of other sequences do not move."""
    hq, hkv, d, group, bs = 8, 2, 128, 64, 16
    q, cache, tables, ctx, last = batch([200, 3000, 90], [64, 20, 90], hq, hkv, d, group, bs, 55)
    for bad in (cache.shape[0], -1, 2**31 - 1):
        spoilt, zero = tables.clone(), tables.clone()
        spoilt[1, 7], zero[1, 7] = bad, 0
        out = kops.prefill_attention_kv4(q, cache, spoilt, ctx, last, 0.1, bs)
        assert kops.check_status() == 3
        assert torch.equal(out, kops.prefill_attention_kv4(q, cache, zero, ctx, last, 0.1, bs))
        assert kops.check_status() == 0

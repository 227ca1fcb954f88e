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

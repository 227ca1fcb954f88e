"""The paged cache held in 4 bits on the CPU: its format, and its operators' plain forms."""

import math

import pytest
import torch

from everserve_b200.ops import ref


@pytest.mark.parametrize("d,group", [(64, 64), (128, 64), (128, 128)])
def test_format(d, group):
    """Each channel of a row where the format says it is, from the bytes one at a time."""
    bs, hkv, nb = 16, 2, 3
    g = torch.Generator().manual_seed(d + group)
    cache = torch.zeros(ref.kv4_cache_shape(nb, hkv, bs, d, group), dtype=torch.uint8)
    qkv = torch.randn(2, 3 * hkv * d, generator=g)
    pos, slots = torch.tensor([5, 9]), torch.tensor([bs + 3, -1])
    cs = ref.cos_sin_table(d, 32, 1e4)
    q = ref.rope_kv4_write(qkv, None, pos, cs, slots, cache, hkv, hkv, bs)
    dense = torch.zeros(nb, 2, hkv, bs, d)
    assert torch.equal(q, ref.rope_kv_write(qkv, None, pos, cs, slots, dense, hkv, hkv, bs))
    k, v = ref.kv4_read(cache, slots, d, bs)
    assert not bool(k[1].any()) and not bool(v[1].any())
    assert not bool(cache[0].any()) and not bool(cache[2].any())
    for side, got in ((0, k), (1, v)):
        for h in range(hkv):
            rec = cache[1, h].tolist()
            x = dense[1, side, h, 3].double()
            for c in range(d):
                word = 2 * (c // 8 % 8) + c // 64 if d == 128 else c // 8
                bit = 4 * (c % 8 // 2) + 16 * (c % 2)
                byte = rec[side * bs * d // 2 + 3 * d // 2 + 4 * word + bit // 8]
                code = byte >> 4 if bit % 8 else byte & 15
                at = bs * d + side * bs * 4 * (d // group) + 3 * 4 * (d // group) + 4 * (c // group)
                scale, zero = torch.tensor(rec[at : at + 4], dtype=torch.uint8).view(torch.bfloat16).double().tolist()
                part = x[c // group * group :][:group]
                assert abs(zero - float(part.min())) <= abs(float(part.min())) * 2.0**-8
                assert abs(scale - float(part.max() - part.min()) / 15) <= scale * 2.0**-7
                assert abs(code * scale + zero - float(got[0, h, c])) <= 1e-5
                assert abs(float(got[0, h, c]) - float(x[c])) <= 0.5 * scale + 15 * scale * 2.0**-8 + abs(zero) * 2.0**-8


def test_equal_and_not_finite_groups():
    x = torch.full((4, 64), 1.5)
    x[1, 3], x[2, 4], x[3, 5] = math.nan, math.inf, -math.inf
    c, p = ref.kv4_quantize(x, 1)
    y = ref.kv4_values(c, p.flatten(-2).contiguous().view(torch.uint8))
    assert torch.equal(y[0], x[0]) and bool(y[1:].isnan().all())


def test_shapes_refused():
    for bad in ((2, 1, 16, 96, 64), (2, 1, 8, 64, 64), (2, 1, 16, 128, 32), (2, 1, 16, 64, 128)):
        with pytest.raises(ValueError):
            ref.kv4_cache_shape(*bad)
    with pytest.raises(ValueError):
        ref.kv4_groups(torch.zeros(2, 1, 100, dtype=torch.uint8), 64, 16)


def test_attention_plain_form():
    """The plain attention on a cache in 4 bits is the dense cache's attention on the values held."""
    from everserve_b200.ops import RefOps

    ops, bs, hkv, d, hq = RefOps("cpu"), 16, 2, 64, 4
    g = torch.Generator().manual_seed(3)
    cache = torch.zeros(ref.kv4_cache_shape(9, hkv, bs, d), dtype=torch.uint8)
    slots = torch.randperm(9 * bs, generator=g)
    qkv = torch.randn(9 * bs, 8 * d, generator=g)
    ops.rope_kv4_write(qkv, None, slots % 50, ref.cos_sin_table(d, 64, 1e4), slots, cache, hq, hkv, bs)
    dense = ref.kv4_cache_values(cache, d, bs)
    tables = torch.tensor([[3, 1, 7], [0, 5, 2], [4, 6, 8]], dtype=torch.int32)
    ctx = torch.tensor([40, 0, 17], dtype=torch.int32)
    q = torch.randn(3, hq, d, generator=g)
    a = ops.decode_attention_kv4(q, cache, tables, ctx, 0.2, bs)
    b = ref.paged_attention(q[[0, 2]], dense, tables, ctx, torch.tensor([0, 2]), torch.tensor([39, 16]), 0.2)
    torch.testing.assert_close(a[[0, 2]], b, rtol=1e-5, atol=1e-5)
    assert not bool(a[1].any())
    q = torch.randn(12, hq, d, generator=g)
    ctx = torch.tensor([40, 5, 17], dtype=torch.int32)
    a = ops.prefill_attention_kv4(q, cache, tables, ctx, torch.tensor([6, 8, 11]), 0.2, bs)
    seq = torch.tensor([0] * 7 + [1] * 2 + [2] * 3)
    pos = torch.tensor(list(range(33, 40)) + [3, 4, 14, 15, 16])
    torch.testing.assert_close(a, ref.paged_attention(q, dense, tables, ctx, seq, pos, 0.2), rtol=1e-5, atol=1e-5)


def test_copy_pages_pairs():
    from everserve_b200.ops import RefOps

    ops = RefOps("cpu")
    cache = torch.arange(12.0).view(4, 3)
    ops.copy_pages([cache], torch.tensor([[0, 2], [-1, 1], [1, 3]]))
    assert cache[:, 0].tolist() == [0, 3, 0, 3]
    for bad in ([[0, 1], [2, 1]], [[0, 1], [1, 2]], [[2, 2]]):
        with pytest.raises(ValueError):
            ops.copy_pages([cache], torch.tensor(bad))


def test_not_finite_values_reach_the_rows_that_see_them():
    """A group of V that reads as NaN makes its channels of the rows that see the key NaN, and no other."""
    d, bs, n = 128, 16, 20
    g = torch.Generator().manual_seed(4)
    cache = torch.zeros(ref.kv4_cache_shape(2, 1, bs, d), dtype=torch.uint8)
    qkv = torch.randn(n, 4 * d, generator=g)
    tables, ctx, last = torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([n], dtype=torch.int32), torch.tensor([n - 1])

    def attend():
        at = torch.arange(n)
        q = ref.rope_kv4_write(qkv, None, at, ref.cos_sin_table(d, 32, 1e4), at, cache, 2, 1, bs)
        return ref.kv4_attention(q, cache, tables, ctx, last, 0.1, bs)

    want = attend()
    qkv[17, -1] = math.inf  # V's second group
    got = attend()
    bad = torch.zeros(n, 2, d, dtype=torch.bool)
    bad[17:, :, 64:] = True
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad])


def test_a_lost_page_shows():
    """What the device tests allow over long histories (0.28 % of the norm) is far less than a page of 16 keys in
    5,000 missing from the definition, or operands of 8 bits, cost."""
    g = torch.Generator().manual_seed(6)
    n, t, d = 5000, 16, 128
    q, v = torch.randn(t, d, generator=g).double(), torch.randn(n, d, generator=g).double()
    k = (torch.randn(n, d, generator=g) + 2 * torch.randn(d, generator=g)).double()

    def attend(k, v, round_p=False):
        p = torch.softmax(q @ k.T * d**-0.5, -1)
        return (p.bfloat16().double() if round_p else p) @ v

    want = attend(k, v)
    lost = torch.cat([torch.arange(2000), torch.arange(2016, n)])
    for got in (attend(k[lost], v[lost]), attend(k.bfloat16().double(), v.bfloat16().double(), True)):
        assert float((got - want).norm() / want.norm()) > 0.0028


def test_what_a_group_holds():
    """A value is held within half a stored scale or, far from zero, within what rounding the pair to bf16 moves the
    group's ends by: 2^-8 of its smallest value and of its range. A range past fp32's largest number reads as NaN."""
    g = torch.Generator().manual_seed(7)
    for offset in (0.0, -1.0, 10.0, 100.0, -3000.0, 1e30):
        for spread in (1.0, 0.1):
            x = torch.randn(200, 64, generator=g) * spread * max(1.0, abs(offset) / 100) + offset
            c, p = ref.kv4_quantize(x, 1)
            held = ref.kv4_values(c, p.flatten(-2).contiguous().view(torch.uint8)).double()
            low, high = x.amin(-1, keepdim=True).double(), x.amax(-1, keepdim=True).double()
            ends = 2.0**-8 * (low.abs() + (high - low))
            tol = torch.maximum(0.5 * p[..., 0].double(), ends) * (1 + 1e-4) + 2.0**-22 * (high.abs() + low.abs())
            assert bool(((held - x.double()).abs() <= tol).all())
    x = torch.zeros(3, 64)
    x[0, 0], x[0, 1] = 3e38, -3e38
    x[1, 0], x[1, 1] = 1.6e38, -1.6e38
    c, p = ref.kv4_quantize(x, 1)
    y = ref.kv4_values(c, p.flatten(-2).contiguous().view(torch.uint8))
    assert bool(y[0].isnan().all()) and bool(torch.isfinite(y[1:]).all())

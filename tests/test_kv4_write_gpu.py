"""Writes of the paged cache held in 4 bits whose arguments are out of range."""

import pytest
import torch

from everserve_b200.ops import KernelOps, ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return KernelOps("cuda:0")


@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32)])
def test_a_bad_position_writes_nothing(kops, d, bs):
    """The row of a position outside the table is reported and not written, though its slot is one; the
    step's other rows are."""
    hq, hkv = 4, 2
    cs = ref.cos_sin_table(d, 64, 1e4).cuda()
    qkv = torch.randn(3, (hq + 2 * hkv) * d, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    slots = torch.tensor([1, 2, 3], device="cuda")
    assert kops.check_status() == 0
    for bad in (64, -1):
        cache = torch.full(ref.kv4_cache_shape(2, hkv, bs, d), 0xA5, dtype=torch.uint8, device="cuda")
        want = cache.clone()
        pos = torch.tensor([7, bad, 9], device="cuda")
        kops.rope_kv4_write(qkv, None, pos, cs, slots, cache, hq, hkv, bs)
        assert kops.check_status() == 3
        ref.rope_kv4_write(qkv[::2], None, pos[::2], cs, slots[::2], want, hq, hkv, bs)
        assert torch.equal(cache, want)


@pytest.mark.parametrize("d,group,bs", [(64, 64, 16), (128, 64, 16), (128, 128, 32)])
def test_wide_ranges_and_far_offsets(kops, d, group, bs):
    """Groups far from zero, of ranges near fp32's largest number and past it (which read as NaN): byte for byte the
    format's formula."""
    hq, hkv, n = 2, 2, 12
    x = torch.randn(n, hq + 2 * hkv, d, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    for i, off in enumerate((0, 10, -100, 3000, 1e30, -1e-30)):
        x[i] += off
    x[6] *= 1e38 / 4
    x[7] *= 1e-37
    x[8, -1, 0], x[8, -1, 1] = 3e38, -3e38
    x[9, -1, d - 1], x[9, -1, d - 2] = 1.6e38, -1.6e38
    qkv = x.bfloat16().flatten(1)
    cs = ref.cos_sin_table(d, 64, 1e4).cuda()
    pos, slots = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.arange(n, device="cuda")  # no rotation
    cache = torch.zeros(ref.kv4_cache_shape(1, hkv, bs, d, group), dtype=torch.uint8, device="cuda")
    want = cache.clone()
    kops.rope_kv4_write(qkv, None, pos, cs, slots, cache, hq, hkv, bs)
    ref.rope_kv4_write(qkv, None, pos, cs, slots, want, hq, hkv, bs)
    assert torch.equal(cache, want) and kops.check_status() == 0
    _, v = kops.kv4_read(cache, slots, d, bs)
    bad = torch.zeros(n, hkv, d, dtype=torch.bool, device="cuda")
    bad[8, -1, :group] = True
    assert torch.equal(v.isnan(), bad)

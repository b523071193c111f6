"""Products of few rows that need more workgroups than one launch holds (2^22 of sixteen columns)."""
import pytest
import torch

import ctc_amd
from tests import scaled_reference as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def bounded(got, want, mag, k, dtype):
    assert bool(((got.double() - want).abs() <= ref.product_bound(want, mag, k, dtype)).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_entries_of_few_rows(cuda, dtype):
    """65535 entries of 1040 columns: 65 * 65535 workgroups."""
    g = torch.Generator().manual_seed(1)
    batch, n, k = 65535, 1040, 24
    A, sa = ref.random_operand(g, (batch, 1, k), "rows")
    B, sb = ref.random_operand(g, (n, k), "tiles")
    frame = torch.full((batch, 2, n), 5.0, dtype=dtype, device="cuda")
    launches = ctc_amd.get_option("launches_scaled_skinny")
    ctc_amd.scaled_contract(A, sa, B.expand(batch, n, k), sb.expand(batch, *sb.shape), out=frame[:, :1], alpha=0.5)
    assert ctc_amd.get_option("launches_scaled_skinny") == launches + 1
    want, mag = ref.product(A[:, 0], sa[:, 0], B, sb)
    bounded(frame[:, 0], 0.5 * want, 0.5 * mag, k, dtype)
    assert bool((frame[:, 1] == 5).all())


def test_many_groups_of_few_rows(cuda):
    """65535 groups, most of them empty, of 1040 columns; the rows in front of the first and behind the last stay as they are."""
    g = torch.Generator().manual_seed(2)
    groups, n, k = 65535, 1040, 136
    counts = torch.zeros(groups, dtype=torch.int64)
    for e, c in ((0, 3), (1, 20), (30000, 1), (64511, 40), (64512, 2), (65534, 17)):
        counts[e] = c
    rows = 2 + int(counts.sum()) + 3
    A, sa = ref.random_operand(g, (rows, k), "rows")
    B, sb = ref.random_operand(g, (n, k), "tiles")
    scale = sb.expand(groups, *sb.shape) * torch.exp2(torch.arange(groups, device="cuda") % 4.0)[:, None, None]
    off = torch.cat([torch.tensor([2]), 2 + counts.cumsum(0)]).to(torch.int32).cuda()
    out = torch.full((rows, n), 5.0, device="cuda")
    ctc_amd.scaled_grouped_contract(A, sa, B.expand(groups, n, k), scale, off, out=out)
    assert bool((out[:2] == 5).all()) and bool((out[-3:] == 5).all())
    at = 2
    for e in counts.nonzero()[:, 0].tolist():
        end = at + int(counts[e])
        want, mag = ref.product(A[at:end], sa[at:end], B, sb * 2.0 ** (e % 4))
        bounded(out[at:end], want, mag, k, F32)
        at = end


@pytest.mark.parametrize("block", ["tiles", "rows"])
def test_more_columns_than_one_launch_holds(cuda, block):
    g = torch.Generator().manual_seed(3)
    n, k = 16 * 0x3fffff + 2000, 16
    A, sa = ref.random_operand(g, (2, k), "rows")
    codes = torch.randint(0, 0x7F, (n, k), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    B = codes.view(torch.float8_e4m3fn)
    r = ref.cdiv(n, 128) if block == "tiles" else n
    sb = torch.exp2(torch.arange(r, device="cuda") % 7.0 - 6)[:, None]
    got = ctc_amd.scaled_contract(A, sa, B, sb)
    for at in range(0, n, 1 << 24):  # in pieces of whole tiles
        end = min(n, at + (1 << 24))
        part = sb[at // 128:ref.cdiv(end, 128)] if block == "tiles" else sb[at:end]
        want, mag = ref.product(A, sa, B[at:end], part)
        bounded(got[:, at:end], want, mag, k, BF16)

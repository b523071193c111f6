"""Block-scaled products over the whole range of their f32 scales: the two scales of a block may multiply to less than the smallest
normal number or to more than the largest one while the result is an ordinary f32 number."""
import pytest
import torch

import ctc_amd
from tests import scaled_reference as ref

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BF16, F32 = torch.bfloat16, torch.float32
SUBNORMAL_STEP = {BF16: 2.0 ** -133, F32: 2.0 ** -149}
# powers of two of the scales of successive rows (or tiles of rows): the quantiser's smallest are 2^-109 (e4m3) and 2^-116 (e5m2),
# its largest 2^120; a caller's own may be any f32 number
A_POWERS = (-109, 0, 64, -149, 120, -30, -80, 100, -116, 126, 30, -140)
B_POWERS = (-30, 100, 0, -109, 64, -60, 126, -149, 119)


def wide_scales(scale, powers, g):
    """Scales that stay within a factor of two along a row and step through `powers` from row to row."""
    n = scale.shape[-2]
    p = torch.tensor(powers, dtype=torch.float64)[torch.arange(n) % len(powers)][:, None]
    m = 1 + torch.rand(scale.shape, generator=g, dtype=torch.float64)
    return (m * torch.exp2(p)).float().to(scale.device)


def operand(g, shape, block, powers, dtype=E4M3, pitch=None):
    q, s = ref.random_operand(g, shape, block, dtype, pitch=pitch)
    q.view(torch.uint8)[..., 4::5, :] = 0  # whole rows of zeros, under every scale
    return q, wide_scales(s, powers, g)


def check(A, sa, B, sb, got, dtype, k0=0, k1=None):
    """Where the magnitudes' sum is an f32 number: the bound of ref.product_bound, its last term the subnormal steps (one for each
    block and sum, and one for the result's type).  A row or column of zeros gives zeros whatever its scale."""
    want, mag = ref.product(A, sa, B, sb, k0, k1)
    k = A.shape[-1] if k1 is None else k1 - k0
    fast = dtype is BF16 and A.shape[-2] > 32
    bound = ref.product_bound(want, mag, k, dtype, fast=fast) - 1e-37 + (ref.cdiv(k, 128) + 64) * 2.0 ** -147 + SUBNORMAL_STEP[dtype]
    sure = mag < 2.0 ** 126
    err = (got.double() - want).abs()
    bad = sure & ~(err <= bound)
    assert not bool(bad.any()), "%d of %d off, first at %s" % (int(bad.sum()), int(sure.sum()), bad.nonzero()[0].tolist())
    assert bool((mag[sure] > 2.0 ** -126).any()) and bool((mag == 0).any())


@pytest.mark.parametrize("m, n, k", [
    (5, 1000, 400), (20, 1200, 384), (3, 20000, 272),  # rows straight to registers: eight waves, two row tiles, two waves
    (150, 1200, 400), (150, 1100, 301), (150, 600, 4096), (150, 600, 4099),  # few tiles: DMA, registers, K split
    (2048, 2304, 272), (2048, 2304, 301),  # more tiles than compute units
    (4096, 4096, 272), (2304, 8192, 144), (2100, 8192, 272),  # large tiles, halves, light ones
])
@pytest.mark.parametrize("blocks", [("rows", "tiles"), ("rows", "rows"), ("tiles", "rows")])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("a_dtype", [E4M3, E5M2])
def test_product_over_the_scales_range(cuda, m, n, k, blocks, dtype, a_dtype):
    g = torch.Generator().manual_seed(m + n + k)
    A, sa = operand(g, (m, k), blocks[0], A_POWERS, a_dtype)
    B, sb = operand(g, (n, k), blocks[1], B_POWERS)
    check(A, sa, B, sb, ctc_amd.scaled_contract(A, sa, B, sb, dtype=dtype), dtype)


@pytest.mark.parametrize("counts", [[3, 0, 5, 4], [300, 0, 128, 700], [2304, 100]])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_groups_of_rows_over_the_scales_range(cuda, counts, dtype):
    g = torch.Generator().manual_seed(sum(counts))
    n = 8192 if sum(counts) > 2000 else 1100
    A, sa = operand(g, (sum(counts), 400), "rows", A_POWERS)
    B, sb = operand(g, (n, 400), "tiles", B_POWERS)
    off = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    got = ctc_amd.scaled_grouped_contract(A, sa, B.expand(len(counts), n, 400), sb.expand(len(counts), *sb.shape), off, dtype=dtype)
    check(A, sa, B, sb, got, dtype)


@pytest.mark.parametrize("m, n", [(150, 300), (2304, 2048)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_groups_of_the_contracted_index_over_the_scales_range(cuda, m, n, dtype):
    g = torch.Generator().manual_seed(m)
    A, sa = operand(g, (m, 900), "rows", A_POWERS, E5M2)
    B, sb = operand(g, (n, 900), "rows", B_POWERS)
    at = [0, 256, 256, 640, 900]
    got = ctc_amd.scaled_grouped_contract(A, sa, B, sb, torch.tensor(at, dtype=torch.int32, device="cuda"), along="contracted", dtype=dtype)
    for e in range(4):
        if at[e + 1] > at[e]:
            check(A, sa, B, sb, got[e], dtype, at[e], at[e + 1])
    assert bool((got[1] == 0).all())


@pytest.mark.parametrize("m", [6, 150, 2304])
def test_blocks_of_the_quantizer_at_both_ends_of_its_range(cuda, m):
    """All-zero rows carry the floor's scale; rows near f32's largest number meet columns of zeros and of tiny values, and of large
    ones that are zero where the row is not."""
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, 400, generator=g)
    x[::3] *= 1e37 / x[::3].abs().amax()
    x[1::3] = 0
    x[::6, 1:] = 0
    x[::6, 0] = 1e37
    w = torch.randn(2048, 400, generator=g)
    w[:500] = 0
    w[500:1000] *= 1e38 / w[500:1000].abs().amax()
    w[500:700, 0] = 0
    w[1000:1500] *= 1e-36
    qx, sx = ctc_amd.block_quantize(x.cuda())
    qw, sw = ctc_amd.block_quantize(w.cuda(), "rows")
    for dtype in (F32, BF16):
        check(qx, sx, qw, sw, ctc_amd.scaled_contract(qx, sx, qw, sw, dtype=dtype), dtype)


def test_ordinary_blocks_keep_their_bits_beside_extreme_ones(cuda):
    """Rows and columns of ordinary scales give the same bits whatever scales the others in their tile carry."""
    g = torch.Generator().manual_seed(7)
    for m, k in ((20, 400), (150, 400), (150, 301), (2304, 400)):
        A, sa = ref.random_operand(g, (m, k), "rows")
        B, sb = ref.random_operand(g, (2048, k), "rows")
        for dtype in (F32, BF16):
            want = ctc_amd.scaled_contract(A, sa, B, sb, dtype=dtype)
            ta, tb = sa.clone(), sb.clone()
            ta[1::2] = 2.0 ** -120
            tb[1::2] = 2.0 ** 120
            got = ctc_amd.scaled_contract(A, ta, B, tb, dtype=dtype)
            assert torch.equal(got[::2, ::2], want[::2, ::2])

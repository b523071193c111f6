"""Block-scaled 8-bit operators against their definitions in 64 bits."""
import pytest
import torch

import ctc_amd
from tests import scaled_reference as ref

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def same_codes(got, want):
    """Equal 8-bit codes; any NaN equals any other."""
    g, w = got.cpu().contiguous().view(torch.uint8).reshape(-1), want.contiguous().view(torch.uint8).reshape(-1)
    gn, wn = got.cpu().float().isnan().reshape(-1), want.float().isnan().reshape(-1)
    assert torch.equal(gn, wn)
    assert torch.equal(g[~gn], w[~wn])


def strided(x, pad, shift):
    """The same values with rows `pad` further apart, `shift` elements into an allocation."""
    *lead, r, c = x.shape
    n = 1
    for d in lead:
        n *= d
    flat = torch.full((n * r * (c + pad) + shift,), float("nan"), dtype=x.dtype, device="cuda")
    v = flat[shift:].reshape(*lead, r, c + pad)[..., :c]
    v.copy_(x)
    return v


# ---- quantiser ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("block", ["rows", "tiles"])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("src", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 127), (128, 128), (129, 257), (300, 1000), (257, 8), (2, 130, 200), (1, 65, 129)])
def test_quantizer(cuda, block, dtype, src, shape):
    x = torch.randn(shape, generator=gen(1)) * torch.exp2(torch.randint(-20, 20, shape[-1:], generator=gen(2)).float())
    x = x.to(src).cuda()
    q, s, qt, st = ctc_amd.block_quantize(x, block, dtype, transposed="both")
    wq, ws = ref.quantize(x, block, dtype)
    wqt, wst = ref.quantize(x.transpose(-1, -2), block, dtype)
    same_codes(q, wq)
    same_codes(qt, wqt)
    assert torch.equal(s.cpu(), ws) and torch.equal(st.cpu(), wst)
    assert torch.equal(ctc_amd.block_quantize(x, block, dtype)[0].cpu().view(torch.uint8), q.cpu().view(torch.uint8))
    assert len(ctc_amd.block_quantize(x, block, dtype, transposed=1)) == 2
    one = ctc_amd.block_quantize(x, block, dtype, transposed=True)
    same_codes(one[0], wqt)
    assert torch.equal(one[1].cpu(), wst)


@pytest.mark.parametrize("src", [F32, BF16])
@pytest.mark.parametrize("pad, shift", [(0, 0), (1, 0), (3, 1), (8, 5)])
@pytest.mark.parametrize("transposed", [False, "both"])
def test_quantizer_strides_and_results_in_place(cuda, src, pad, shift, transposed):
    x = strided(torch.randn(2, 150, 321, generator=gen(3)).to(src), pad, shift)
    # results inside larger tensors: nothing around them changes
    frames = [torch.full((2, 150 + 2, 321 + 7), 0x55, dtype=torch.uint8, device="cuda"), torch.full((2, 321 + 2, 150 + 5), 0x55, dtype=torch.uint8, device="cuda")]
    views = [frames[0][:, 1:151, 3:324].view(E4M3), frames[1][:, 1:322, 2:152].view(E4M3)]
    scales = [torch.full((2, 150, 3 + 2), -7.0, device="cuda"), torch.full((2, 321, 2 + 2), -7.0, device="cuda")]
    out = []
    for i in range(2 if transposed == "both" else 1):
        out += [views[i], scales[i][..., 1:-1]]
    got = ctc_amd.block_quantize(x, "rows", E4M3, transposed=transposed, out=out)
    for i, y in enumerate([x, x.transpose(-1, -2)][: len(out) // 2]):
        wq, ws = ref.quantize(y, "rows", E4M3)
        same_codes(got[2 * i], wq)
        assert torch.equal(got[2 * i + 1].cpu(), ws)
        edge = frames[i].clone()
        edge[:, 1:1 + wq.shape[1], (3, 2)[i]:(3, 2)[i] + wq.shape[2]] = 0x55
        assert bool((edge == 0x55).all())
        assert bool((scales[i][..., 0] == -7).all()) and bool((scales[i][..., -1] == -7).all())


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("block", ["rows", "tiles"])
def test_quantizer_special_values(cuda, dtype, block):
    x = torch.randn(130, 400, generator=gen(4))
    x[0, 5] = float("nan")
    x[1, 200] = float("inf")
    x[2, 201] = float("-inf")
    x[3] = 0
    x[4, :128] = -0.0
    x[5] = 1e-40
    x[6, 100] = torch.finfo(torch.float32).max
    x[7] = torch.finfo(torch.float32).tiny
    x[129, 256:] = float("nan")
    x = x.cuda()
    q, s, qt, st = ctc_amd.block_quantize(x, block, dtype, transposed="both")
    for got, scale, y in ((q, s, x), (qt, st, x.t())):
        wq, ws = ref.quantize(y, block, dtype)
        same_codes(got, wq)
        assert torch.equal(scale.cpu(), ws)
        assert bool(scale.isfinite().all()) and bool((scale > 0).all())


def test_quantizer_error_is_half_a_step(cuda):
    """|x - q scale| <= 2^-4 |x| (e4m3) above the type's smallest normal number, half its subnormal step below; f32 roundings of
    the quotients and the product add 4 * 2^-24 of the value."""
    x = torch.randn(200, 700, generator=gen(5)).cuda()
    q, s = ctc_amd.block_quantize(x)
    back = ref.values(q, s)
    step = ref.spread(s, 200, 700) * 2.0 ** -10  # half of 2^-9
    bound = torch.maximum(x.double().abs() * 2.0 ** -4, step) * (1 + 2.0 ** -18) + x.double().abs() * 4 * 2.0 ** -24
    assert bool(((back - x.double()).abs() <= bound).all())


# ---- products --------------------------------------------------------------------------------------------------------
def check_product(A, sa, B, sb, got, dtype, alpha=1.0, beta=0.0, before=None, fast=None):
    """fast: the product may sum with the matrix core's 8-bit form (bf16 results of more than 32 rows)."""
    fast = dtype is BF16 and (A.shape[-2] > 32 if fast is None else fast)
    want, mag = ref.product(A, sa, B, sb)
    want = alpha * want
    if beta:
        want = want + beta * before.double()
    bound = ref.product_bound(want, mag, A.shape[-1], dtype, alpha, beta, None if before is None else before.double(), fast)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), "off by %.3g of the bound" % float((err / bound).max())


SIZES = [
    (1, 1, 1), (1, 16, 128), (1, 1000, 2048), (2, 17, 129), (15, 300, 1111), (16, 64, 4096), (17, 130, 256), (32, 48, 640), (33, 40, 100),
    (64, 1, 128), (100, 129, 127), (128, 128, 128), (129, 255, 400), (200, 300, 16384), (256, 256, 256), (300, 520, 1040), (1000, 17, 33),
]


@pytest.mark.parametrize("m, n, k", SIZES)
@pytest.mark.parametrize("blocks", [("rows", "tiles"), ("rows", "rows"), ("tiles", "tiles"), ("tiles", "rows")])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_product(cuda, m, n, k, blocks, dtype):
    g = gen(m * 7 + n * 3 + k)
    A, sa = ref.random_operand(g, (m, k), blocks[0])
    B, sb = ref.random_operand(g, (n, k), blocks[1])
    check_product(A, sa, B, sb, ctc_amd.scaled_contract(A, sa, B, sb, dtype=dtype), dtype)


@pytest.mark.parametrize("m, n, k", [(1, 130, 300), (20, 130, 300), (130, 140, 400), (2049, 4099, 272)])
def test_product_e5m2(cuda, m, n, k):
    g = gen(m)
    A, sa = ref.random_operand(g, (m, k), "rows", E5M2)
    B, sb = ref.random_operand(g, (n, k), "tiles")
    check_product(A, sa, B, sb, ctc_amd.scaled_contract(A, sa, B, sb, dtype=F32), F32)


@pytest.mark.parametrize("m, n, k", [(4096, 4096, 128), (4096, 4096, 528), (3841, 4000, 1032), (2048, 8192, 257), (5000, 3500, 640)])
@pytest.mark.parametrize("blocks", [("rows", "tiles"), ("rows", "rows")])
def test_product_large(cuda, m, n, k, blocks):
    g = gen(k)
    pitch = ref.cdiv(k, 16) * 16
    A, sa = ref.random_operand(g, (m, k), blocks[0], pitch=pitch)
    B, sb = ref.random_operand(g, (n, k), blocks[1], pitch=pitch)
    before = ctc_amd.get_option("launches_scaled_256")
    got = ctc_amd.scaled_contract(A, sa, B, sb)
    assert ctc_amd.get_option("launches_scaled_256") == before + 1
    check_product(A, sa, B, sb, got, BF16)


# On 256 compute units: full tiles alone, a last round in halves, a light last row, both, several entries, light tiles alone
@pytest.mark.parametrize("batch, m, n, k", [
    (1, 2048, 8192, 144), (1, 2304, 8192, 160), (1, 2100, 8192, 400), (1, 2400, 8200, 272), (3, 1500, 4000, 16), (2, 1400, 5000, 656), (1, 100, 60000, 144),
    (1, 129, 60000, 1296),
])
@pytest.mark.parametrize("blocks", [("rows", "tiles"), ("tiles", "rows")])
@pytest.mark.parametrize("a_dtype", [E4M3, E5M2])
def test_product_in_full_tiles_halves_and_light_tiles(cuda, batch, m, n, k, blocks, a_dtype):
    g = gen(m + n + k)
    A, sa = ref.random_operand(g, (batch, m, k), blocks[0], a_dtype)
    B, sb = ref.random_operand(g, (batch, n, k), blocks[1])
    if a_dtype is E5M2:
        sa = sa * 2.0 ** -7  # e5m2's values reach 2^7 times as far
    whole = torch.randn(batch, m + 2, n, generator=g).to(BF16).cuda()
    before = whole.clone()
    launches = ctc_amd.get_option("launches_scaled_256")
    # every element once: a second visit would add to it again
    ctc_amd.scaled_contract(A, sa, B, sb, out=whole[:, 1:-1], alpha=0.5, beta=0.75)
    assert ctc_amd.get_option("launches_scaled_256") == launches + 1
    assert torch.equal(whole[:, 0], before[:, 0]) and torch.equal(whole[:, -1], before[:, -1])
    for b in range(batch):
        check_product(A[b], sa[b], B[b], sb[b], whole[b, 1:-1], BF16, 0.5, 0.75, before[b, 1:-1])


@pytest.mark.parametrize("m", [1, 20, 150, 2500])
@pytest.mark.parametrize("pitch, shift", [(304, 16), (301, 0), (303, 5), (320, 3), (305, 0)])
def test_product_alignments(cuda, m, pitch, shift):
    """Every pitch and base; the bytes around the elements are NaN codes."""
    g = gen(m + pitch)
    A, sa = ref.random_operand(g, (m, 301), "rows", pitch=pitch, lead_offset=shift)
    B, sb = ref.random_operand(g, (4200, 301), "tiles", pitch=pitch, lead_offset=16)
    check_product(A, sa, B, sb, ctc_amd.scaled_contract(A, sa, B, sb), BF16)


@pytest.mark.parametrize("m, n, k", [(1, 100, 256), (40, 100, 384), (130, 300, 128), (150, 140, 8192)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pad, shift", [(0, 0), (3, 1), (4, 0)])
def test_product_adds_to_a_strided_result(cuda, m, n, k, dtype, pad, shift):
    g = gen(n + k)
    A, sa = ref.random_operand(g, (3, m, k), "rows")
    B, sb = ref.random_operand(g, (3, n, k), "tiles")
    frame = torch.randn(3 * (m + 1) * (n + pad) + shift, generator=g).to(dtype).cuda()
    first = frame.clone()
    out = frame[shift:].reshape(3, m + 1, n + pad)[:, :m, :n]
    before = out.clone()
    got = ctc_amd.scaled_contract(A, sa, B, sb, out=out, alpha=-0.75, beta=1.5)
    assert got is out
    check_product(A, sa, B, sb, out, dtype, -0.75, 1.5, before)
    frame[shift:].reshape(3, m + 1, n + pad)[:, :m, :n] = before
    assert torch.equal(frame, first)


def test_product_without_beta_does_not_read_the_result(cuda):
    g = gen(9)
    for m in (2, 200):
        A, sa = ref.random_operand(g, (m, 256), "rows")
        B, sb = ref.random_operand(g, (300, 256), "tiles")
        out = torch.full((m, 300), float("nan"), device="cuda")
        check_product(A, sa, B, sb, ctc_amd.scaled_contract(A, sa, B, sb, out=out), F32)


@pytest.mark.parametrize("m", [3, 70])
def test_product_of_an_empty_contraction(cuda, m):
    A, sa = torch.empty(m, 0, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(m, 0, device="cuda")
    B, sb = torch.empty(40, 0, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(40, 0, device="cuda")
    assert bool((ctc_amd.scaled_contract(A, sa, B, sb, dtype=F32) == 0).all())
    out = torch.ones(m, 40, device="cuda")
    ctc_amd.scaled_contract(A, sa, B, sb, out=out, beta=2.0)
    assert bool((out == 2).all())
    assert ctc_amd.scaled_contract(A[:0], sa[:0], B, sb).shape == (0, 40)


def test_product_keeps_nan_in_its_row_and_column(cuda):
    g = gen(11)
    for m, n in ((5, 40), (150, 200), (4096, 4096)):
        A, sa = ref.random_operand(g, (m, 384), "rows")
        B, sb = ref.random_operand(g, (n, 384), "tiles")
        A.view(torch.uint8)[3, 200] = 0x7F
        B.view(torch.uint8)[17, 5] = 0x7F
        sa[4, 2] = float("inf")
        got = ctc_amd.scaled_contract(A, sa, B, sb)
        bad = ~got.isfinite()
        assert bool(bad[3].all()) and bool(bad[:, 17].all()) and bool(bad[4].all())
        bad[3] = False
        bad[4] = False
        bad[:, 17] = False
        assert not bool(bad.any())


def test_split_product_is_the_same_every_time(cuda):
    g = gen(12)
    A, sa = ref.random_operand(g, (150, 16384), "rows")
    B, sb = ref.random_operand(g, (260, 16384), "rows")
    before = ctc_amd.get_option("launches_scaled_split")
    first = ctc_amd.scaled_contract(A, sa, B, sb, dtype=F32)
    assert ctc_amd.get_option("launches_scaled_split") == before + 1
    for _ in range(5):
        assert torch.equal(ctc_amd.scaled_contract(A, sa, B, sb, dtype=F32), first)


def test_operands_with_strided_scales_and_a_shared_batch(cuda):
    g = gen(13)
    A, sa = ref.random_operand(g, (2, 70, 300), "rows")
    B, sb = ref.random_operand(g, (90, 300), "tiles")
    wide = torch.zeros(2, 70, 9, device="cuda")
    wide[..., ::3] = sa
    B3, sb3 = B.view(torch.uint8).expand(2, 90, 300).view(E4M3), sb.expand(2, 1, 3)
    got = ctc_amd.scaled_contract(A, wide[..., ::3], B3, sb3, dtype=F32)
    check_product(A, sa, torch.stack([B.view(torch.uint8)] * 2).view(E4M3), torch.stack([sb, sb]), got, F32)


def far(rows, cols, pitch, dtype, values):
    """A rows x cols view whose rows lie `pitch` elements apart: the last one starts beyond 2^32 bytes."""
    assert (rows - 1) * pitch * values.element_size() > 2 ** 32
    t = torch.empty((rows - 1) * pitch + cols, dtype=dtype, device="cuda")
    v = t.as_strided((rows, cols), (pitch, 1))
    v.copy_(values)
    return v


@pytest.mark.parametrize("m", [3, 150])
@pytest.mark.parametrize("pitch", [1 << 22, (1 << 22) + 16, (1 << 22) + 1])
def test_operands_and_results_beyond_32_bit_offsets(cuda, m, pitch):
    """The DMA's 32-bit offsets end at pitches of 2^22: beyond, and at odd ones, the blocks pass through registers."""
    g = gen(14)
    A, sa = ref.random_operand(g, (m, 300), "rows")
    B, sb = ref.random_operand(g, (1100, 300), "tiles")
    wide = far(1100, 300, pitch, torch.uint8, B.view(torch.uint8)).view(E4M3)
    check_product(A, sa, B, sb, ctc_amd.scaled_contract(A, sa, wide, sb), BF16)
    out = far(1100, m, 1 << 20, F32, torch.zeros(1100, m, device="cuda"))
    ctc_amd.scaled_contract(wide, sb, A, sa, out=out)
    check_product(B, sb, A, sa, out, F32)


def test_quantizer_beyond_32_bit_offsets(cuda):
    x = torch.randn(1100, 200, generator=gen(15))
    wide = far(1100, 200, 1 << 20, F32, x.cuda())
    q, s, qt, st = ctc_amd.block_quantize(wide, transposed="both")
    wq, ws = ref.quantize(x, "rows", E4M3)
    same_codes(q, wq)
    assert torch.equal(s.cpu(), ws)
    same_codes(qt, ref.quantize(x.t(), "rows", E4M3)[0])


@pytest.mark.parametrize("m", [5, 140])
def test_product_with_the_batch_between_rows_and_columns(cuda, m):
    g = gen(16)
    A, sa = ref.random_operand(g, (m, 3, 256), "rows")  # [m, batch, k]; its scales [m, batch, blocks]: one for each row of any view
    A = A.transpose(0, 1)
    scale = torch.rand(m, 3, 2, generator=g).cuda().transpose(0, 1)
    B, sb = ref.random_operand(g, (3, 60, 256), "tiles")
    out = torch.full((m, 3, 64), 5.0, device="cuda")
    ctc_amd.scaled_contract(A, scale, B, sb, out=out.transpose(0, 1)[..., :60])
    check_product(A, scale, B, sb, out.transpose(0, 1)[..., :60], F32)
    assert bool((out[..., 60:] == 5).all())


# ---- groups ----------------------------------------------------------------------------------------------------------
def offsets_of(counts, first=0):
    return torch.tensor([first] + counts, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


ROW_GROUPS = [
    [1], [0, 5, 0, 1], [16, 17, 1, 0, 33], [300, 0, 1, 128, 129], [0, 0, 0], [700] + [0] * 70 + [3], [2] * 100, [1500, 20, 900, 0, 1300, 4000],
]


@pytest.mark.parametrize("counts", ROW_GROUPS)
@pytest.mark.parametrize("n, k", [(40, 100), (256, 512), (530, 1040)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_groups_of_rows(cuda, counts, n, k, dtype):
    g = gen(sum(counts) + n)
    first, behind = 2, 3
    rows = first + sum(counts) + behind
    A, sa = ref.random_operand(g, (rows, k), "rows")
    B, sb = ref.random_operand(g, (len(counts), n, k), "tiles")
    out = torch.full((rows, n), 5.0, dtype=dtype, device="cuda")
    off = offsets_of(counts, first)
    ctc_amd.scaled_grouped_contract(A, sa, B, sb, off, out=out)
    assert bool((out[:first] == 5).all()) and bool((out[rows - behind:] == 5).all())
    at = off.tolist()
    for e in range(len(counts)):
        if counts[e]:
            lo, hi = at[e], at[e + 1]
            check_product(A[lo:hi], sa[lo:hi], B[e], sb[e], out[lo:hi], dtype, fast=rows > 8 * len(counts))


@pytest.mark.parametrize("counts", [
    [2304], [2304, 100], [128, 129, 256, 257, 384, 385, 1, 0, 2000], [100] * 20, [512] * 5 + [0] * 70 + [130], [3, 2800, 5], [1] * 100 + [1500],
])
@pytest.mark.parametrize("k", [16, 144, 400, 1040])
def test_groups_of_rows_in_full_tiles_halves_and_light_tiles(cuda, counts, k):
    g = gen(sum(counts) + k)
    rows, n = sum(counts) + 1, 8192
    A, sa = ref.random_operand(g, (rows, k), "rows")
    B, sb = ref.random_operand(g, (1, n, k), "tiles")
    B, sb = B.expand(len(counts), n, k), sb * torch.exp2(torch.arange(len(counts), device="cuda") % 5.0)[:, None, None]
    out = torch.randn(rows, n, generator=g).to(BF16).cuda()
    before = out.clone()
    off = offsets_of(counts)
    launches = ctc_amd.get_option("launches_scaled_256")
    ctc_amd.scaled_grouped_contract(A, sa, B, sb, off, out=out, alpha=0.5, beta=0.75)
    assert ctc_amd.get_option("launches_scaled_256") == launches + 1
    assert torch.equal(out[-1], before[-1])
    at = off.tolist()
    for e in range(len(counts)):
        lo, hi = at[e], at[e + 1]
        if hi > lo:
            check_product(A[lo:hi], sa[lo:hi], B[e], sb[e], out[lo:hi], BF16, 0.5, 0.75, before[lo:hi], fast=True)


@pytest.mark.parametrize("blocks", [("rows", "rows"), ("tiles", "tiles")])
@pytest.mark.parametrize("rows", [40, 1000])
def test_groups_of_rows_other_scales(cuda, blocks, rows):
    g = gen(rows)
    A, sa = ref.random_operand(g, (rows, 333), blocks[0], E5M2)
    B, sb = ref.random_operand(g, (5, 200, 333), blocks[1])
    counts = [rows // 2, 0, rows // 4, 1, rows - rows // 2 - rows // 4 - 1]
    off = offsets_of(counts)
    got = ctc_amd.scaled_grouped_contract(A, sa, B, sb, off, dtype=F32, alpha=0.5)
    every = ref.values(A, sa)
    at = off.tolist()
    for e in range(5):
        lo, hi = at[e], at[e + 1]
        b = ref.values(B[e], sb[e])
        want, mag = every[lo:hi] @ b.t().contiguous(), every[lo:hi].abs() @ b.abs().t().contiguous()
        bound = ref.product_bound(0.5 * want, mag, 333, F32, 0.5)
        assert bool(((got[lo:hi].double() - 0.5 * want).abs() <= bound).all())


@pytest.mark.parametrize("bad", [[-5, 3, 10, 10], [0, 8, 4, 10], [0, 5, 2000, 10], [4, 4, 4, 4]])
def test_offsets_outside_the_operands_stay_inside(cuda, bad):
    """Values past the ends count as the ends and a falling pair as an empty group."""
    g = gen(21)
    A, sa = ref.random_operand(g, (10, 256), "rows")
    B, sb = ref.random_operand(g, (3, 100, 256), "tiles")
    frame = torch.full((30, 100), 5.0, device="cuda")
    ctc_amd.scaled_grouped_contract(A, sa, B, sb, torch.tensor(bad, dtype=torch.int32, device="cuda"), out=frame[10:20])
    assert bool((frame[:10] == 5).all()) and bool((frame[20:] == 5).all())
    if bad[0] < 0:
        for e, (lo, hi) in enumerate([(0, 3), (3, 10)]):
            check_product(A[lo:hi], sa[lo:hi], B[e], sb[e], frame[10 + lo:10 + hi], F32)


@pytest.mark.parametrize("counts, tail", [([128], 0), ([256, 0, 128, 384], 0), ([0, 0], 0), ([1024, 128, 0, 0, 256], 128), ([256, 128], 37)])
@pytest.mark.parametrize("m, n", [(1, 7), (100, 130), (300, 257)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_groups_of_the_contracted_index(cuda, counts, tail, m, n, dtype):
    """`tail`: more contracted elements than the groups own, or (37) a last group that ends with K inside a block."""
    g = gen(m + sum(counts))
    if tail == 37:
        counts = counts[:-1] + [counts[-1] + 37]
        k = sum(counts)
    else:
        k = sum(counts) + tail
    A, sa = ref.random_operand(g, (m, k), "rows", E5M2)
    B, sb = ref.random_operand(g, (n, k), "rows")
    off = offsets_of(counts)
    out = torch.full((len(counts), m, n), 3.0, dtype=dtype, device="cuda")
    got = ctc_amd.scaled_grouped_contract(A, sa, B, sb, off, along="contracted", out=out, alpha=0.5, beta=-1.0)
    at = off.tolist()
    for e in range(len(counts)):
        want, mag = ref.product(A, sa, B, sb, at[e], at[e + 1])
        want = 0.5 * want - 3.0
        bound = ref.product_bound(want, mag, counts[e] + 1, dtype, 0.5, -1.0, torch.full_like(want, 3.0), dtype is BF16)
        assert bool(((got[e].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("m, n", [(1100, 2048), (2304, 1024), (1536, 2100), (100, 8000)])
@pytest.mark.parametrize("counts", [[256, 0, 128, 128, 384, 0, 128, 256], [0, 0, 1024, 0, 0, 0, 0, 128]])
def test_groups_of_the_contracted_index_on_the_large_tile(cuda, m, n, counts):
    g = gen(m + n + counts[0])
    k = sum(counts)
    A, sa = ref.random_operand(g, (m, k), "rows")
    B, sb = ref.random_operand(g, (n, k), "rows")
    off = offsets_of(counts)
    out = torch.randn(len(counts), m, n, generator=g).to(BF16).cuda()
    before = out.clone()
    launches = ctc_amd.get_option("launches_scaled_256")
    ctc_amd.scaled_grouped_contract(A, sa, B, sb, off, along="contracted", out=out, alpha=0.5, beta=0.75)
    assert ctc_amd.get_option("launches_scaled_256") == launches + 1
    at = off.tolist()
    for e in range(len(counts)):
        lo, hi = at[e], at[e + 1]
        check_product(A[:, lo:hi], sa[:, lo // 128:hi // 128], B[:, lo:hi], sb[:, lo // 128:hi // 128], out[e], BF16, 0.5, 0.75, before[e], fast=True)


@pytest.mark.parametrize("groups", [64, 65, 200])
def test_many_groups_of_the_contracted_index(cuda, groups):
    """Up to 64 groups the longest come first, beyond that in their order; equal lengths and empty groups among them."""
    g = gen(groups)
    counts = [128 * int(c) for c in torch.randint(0, 4, (groups,), generator=g)]
    k = sum(counts)
    A, sa = ref.random_operand(g, (20, k), "rows")
    B, sb = ref.random_operand(g, (30, k), "rows")
    off = offsets_of(counts)
    got = ctc_amd.scaled_grouped_contract(A, sa, B, sb, off, along="contracted", dtype=F32)
    at = off.tolist()
    for e in range(groups):
        want, mag = ref.product(A, sa, B, sb, at[e], at[e + 1])
        assert bool(((got[e].double() - want).abs() <= ref.product_bound(want, mag, counts[e] + 1, F32)).all())


@pytest.mark.parametrize("bad", [[-300, 128, 256], [256, 128, 512], [0, 1000, 512], [0, 100, 512], [512, 512, 512]])
def test_contracted_offsets_outside_the_operands_stay_inside(cuda, bad):
    """Values past the ends count as the ends, falling pairs as empty and others as the block they fall into."""
    g = gen(22)
    A, sa = ref.random_operand(g, (40, 512), "rows")
    B, sb = ref.random_operand(g, (50, 512), "rows")
    frame = torch.full((4, 40, 50), 5.0, device="cuda")
    ctc_amd.scaled_grouped_contract(A, sa, B, sb, torch.tensor(bad, dtype=torch.int32, device="cuda"), along="contracted", out=frame[1:3])
    assert bool((frame[0] == 5).all()) and bool((frame[3] == 5).all())
    at = [min(max(b, 0), 512) // 128 * 128 for b in bad]
    for e in range(2):
        want, mag = ref.product(A, sa, B, sb, at[e], max(at[e], at[e + 1]))
        assert bool(((frame[1 + e].double() - want).abs() <= ref.product_bound(want, mag, 512, F32)).all())


# ---- the experts' layer -------------------------------------------------------------------------------------------------
def layer_reference(x, up, su, down, sd, pick, gate):
    """(y, bound) in 64 bits.  G x and U x are f32 sums (see product_bound); silu's slope is at most 1.1; exp, the quotient and
    three products add 8 roundings; h is rounded to bf16 once and y once."""
    x, gate = x.double(), gate.double()
    experts, inner = down.shape[0], down.shape[2]
    y = torch.zeros(x.shape[0], down.shape[1], dtype=torch.float64, device=x.device)
    err = torch.zeros_like(y)
    steps = lambda k: (2 * (128 + 2) + ref.cdiv(k, 128) + 16) * ref.F32  # noqa: E731
    for e in range(experts):
        hit = pick == e
        rows = hit.any(1)
        if not bool(rows.any()):
            continue
        w = (gate * hit).sum(1)[rows][:, None]
        u = ref.values(up[e], su[e]).t().contiguous()
        p, pm = x[rows] @ u, x[rows].abs() @ u.abs()
        G, U = p[:, :inner], p[:, inner:]
        dG, dU = (steps(x.shape[1]) * pm).split(inner, 1)
        silu = G * torch.sigmoid(G)
        h = w * silu * U
        dh = w.abs() * (1.1 * dG * (U.abs() + dU) + silu.abs() * dU) + 8 * ref.F32 * h.abs()
        dh = dh + 2.0 ** -8 * (h.abs() + dh)
        d = ref.values(down[e], sd[e]).t().contiguous()
        y[rows] += h @ d
        err[rows] += dh @ d.abs() + steps(inner) * (h.abs() @ d.abs())
    err = err + 2 * experts * ref.F32 * y.abs()
    return y, err + 2.0 ** -8 * (y.abs() + err) + 1e-37


def layer_inputs(seed, tokens, top, experts, hidden, inner):
    g = gen(seed)
    x = torch.randn(tokens, hidden, generator=g).to(BF16).cuda()
    up, su = ref.random_operand(g, (experts, 2 * inner, hidden), "tiles")
    down, sd = ref.random_operand(g, (experts, hidden, inner), "tiles")
    pick = torch.stack([torch.randperm(experts, generator=g)[:top] for _ in range(tokens)]).to(torch.int32).cuda()
    gate = torch.rand(tokens, top, generator=g).cuda()
    # scales of the order that keeps silu in its curved range
    return x, up, su / (100 * hidden ** 0.5) , down, sd, pick, gate


@pytest.mark.parametrize("tokens, top, experts, hidden, inner", [
    (1, 1, 1, 128, 128), (1, 8, 64, 512, 256), (1, 2, 8, 2048, 1024), (2, 1, 3, 130, 70), (5, 3, 7, 100, 33), (16, 2, 4, 256, 384), (17, 4, 60, 384, 144),
    (33, 8, 16, 272, 160), (64, 2, 2, 256, 128), (64, 16, 40, 128, 200), (3, 4, 300, 64, 48), (64, 1, 1, 160, 16),
])
def test_expert_layer(cuda, tokens, top, experts, hidden, inner):
    args = layer_inputs(tokens + top, tokens, top, experts, hidden, inner)
    got = ctc_amd.expert_layer(*args)
    want, bound = layer_reference(*args)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), "off by %.3g of the bound" % float((err / bound).max())
    assert torch.equal(ctc_amd.expert_layer(*args), got)


def test_expert_layer_repeated_and_missing_picks(cuda):
    x, up, su, down, sd, pick, gate = layer_inputs(31, 9, 4, 6, 256, 128)
    pick[0] = torch.tensor([2, 2, 2, 5])
    pick[1] = torch.tensor([-1, 6, 100, 3])
    pick[2] = -1
    pick[8] = 4
    got = ctc_amd.expert_layer(x, up, su, down, sd, pick, gate)
    want, bound = layer_reference(x, up, su, down, sd, pick, gate)
    assert bool(((got.double() - want).abs() <= bound).all())
    assert bool((got[2] == 0).all())


def test_expert_layer_keeps_an_experts_nan_with_its_tokens(cuda):
    x, up, su, down, sd, pick, gate = layer_inputs(32, 20, 2, 5, 256, 128)
    down.view(torch.uint8)[3, :, 7] = 0x7F
    up.view(torch.uint8)[1, 4] = 0x7F
    got = ctc_amd.expert_layer(x, up, su, down, sd, pick, gate)
    hit = ((pick == 3) | (pick == 1)).any(1)
    assert bool(hit.any()) and not bool(hit.all())
    assert bool(got[~hit].isfinite().all())
    assert bool(got[hit].isnan().any(1).all())


def test_expert_layer_strides(cuda):
    x, up, su, down, sd, pick, gate = layer_inputs(33, 6, 3, 8, 200, 96)
    want = ctc_amd.expert_layer(x, up, su, down, sd, pick, gate)
    wide_x = strided(x, 3, 1)
    picks = torch.full((6, 5), 7, dtype=torch.int32, device="cuda")
    gates = torch.full((6, 7), 9.0, device="cuda")
    picks[:, :3], gates[:, :3] = pick, gate
    frame = torch.full((8, 209), 5.0, dtype=BF16, device="cuda")
    ctc_amd.expert_layer(wide_x, up, su, down, sd, picks[:, :3], gates[:, :3], out=frame[1:7, 5:205])
    assert torch.equal(frame[1:7, 5:205], want)
    frame[1:7, 5:205] = 5
    assert bool((frame == 5).all())


# ---- together ---------------------------------------------------------------------------------------------------------
def test_linear_layer_forward_and_gradients(cuda):
    """y = x W^T, dx = dy W, dW = dy^T x from one quantisation of each tensor: the products match the formulas on the
    quantised values, the values match x, W and dy to half a step of e4m3 / e5m2, and a difference quotient of the
    quadratic loss |y - t|^2 / 2 along dx and dW agrees."""
    g = gen(41)
    x = torch.randn(260, 384, generator=g).cuda()
    W = (torch.randn(200, 384, generator=g) * 0.05).cuda()
    t = torch.randn(260, 200, generator=g).cuda()
    qx, sx, qxt, sxt = ctc_amd.block_quantize(x, "rows", transposed="both")
    qw, sw, qwt, swt = ctc_amd.block_quantize(W, "tiles", transposed="both")
    y = ctc_amd.scaled_contract(qx, sx, qw, sw, dtype=F32)
    check_product(qx, sx, qw, sw, y, F32)
    dy = y - t
    qd, sd, qdt, sdt = ctc_amd.block_quantize(dy, "rows", E5M2, transposed="both")
    dx = ctc_amd.scaled_contract(qd, sd, qwt, swt, dtype=F32)
    dW = ctc_amd.scaled_contract(qdt, sdt, qxt, sxt, dtype=F32)
    check_product(qd, sd, qwt, swt, dx, F32)
    check_product(qdt, sdt, qxt, sxt, dW, F32)
    # the transposed tiles are the same values
    assert torch.equal(ref.values(qwt, swt), ref.values(qw, sw).t())
    # against the exact gradients: every product is off by at most half a step of each factor (2^-3 and 2^-4, and their product)
    X, Wd, D = x.double(), W.double(), x.double() @ W.double().t() - t.double()
    noise_y = (2 * 2.0 ** -4 + 2.0 ** -8) * (X.abs() @ Wd.abs().t()) * 1.01 + 1e-6
    # (elements under the smallest normal number: half a subnormal step of their block's scale instead, 2^-10 of 448ths of its top)
    small = lambda a, l: a.abs().amax() * l  # noqa: E731
    noise_y = noise_y + 384 * (small(X, 2.0 ** -10 / 448) * Wd.abs().amax() + small(Wd, 2.0 ** -10 / 448) * X.abs().amax())
    Dabs = D.abs() + noise_y
    sub = Dabs.amax() * 2.0 ** -17 / 57344
    rel = 2.0 ** -3 + 2.0 ** -4 + 2.0 ** -7
    b_dx = noise_y @ Wd.abs() + 1.01 * rel * (Dabs @ Wd.abs()) + 200 * (sub * Wd.abs().amax() + Dabs.amax() * small(Wd, 2.0 ** -10 / 448))
    b_dW = noise_y.t() @ X.abs() + 1.01 * rel * (Dabs.t() @ X.abs()) + 260 * (sub * X.abs().amax() + Dabs.amax() * small(X, 2.0 ** -10 / 448))
    assert bool(((dx.double() - D @ Wd).abs() <= b_dx).all())
    assert bool(((dW.double() - D.t() @ X).abs() <= b_dW).all())
    # differences: the loss is quadratic, so the central quotient is the exact slope (64 bits); the gradients' slope along
    # the same direction is off by at most their bounds' sum along it
    loss = lambda a, b: 0.5 * ((a @ b.t() - t.double()) ** 2).sum()  # noqa: E731
    for grad, bound, vary in ((dx, b_dx, lambda s, v: loss(X + s * v, Wd)), (dW, b_dW, lambda s, v: loss(X, Wd + s * v))):
        v = torch.sign(torch.randn(grad.shape, generator=g)).double().cuda()
        slope = (vary(1e-3, v) - vary(-1e-3, v)) / 2e-3
        assert abs(float((grad.double() * v).sum() - slope)) <= float(bound.sum()) + 1e-5 * abs(float(slope))


def test_expert_layer_agrees_with_grouped_products(cuda):
    """The layer for a few tokens and the path for many (quantised rows, grouped products) give the same result up to the
    quantisation of the activations: the same weights serve both."""
    x, up, su, down, sd, pick, gate = layer_inputs(51, 24, 2, 6, 512, 256)
    want, bound = layer_reference(x, up, su, down, sd, pick, gate)
    order = pick.reshape(-1).argsort(stable=True)
    counts = torch.bincount(pick.reshape(-1).long(), minlength=6)
    off = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    rows = x.repeat_interleave(2, 0)[order]
    q, s = ctc_amd.block_quantize(rows)
    p = ctc_amd.scaled_grouped_contract(q, s, up, su, off, dtype=F32)
    h = torch.nn.functional.silu(p[:, :256]) * p[:, 256:] * gate.reshape(-1)[order][:, None]
    q, s = ctc_amd.block_quantize(h)
    z = ctc_amd.scaled_grouped_contract(q, s, down, sd, off, dtype=F32)
    y = torch.zeros(48, 512, device="cuda")
    y[order] = z
    y = y.reshape(24, 2, 512).sum(1)
    # two quantisations of activations to e4m3: independent relative errors of at most 2^-4 an element; over sums of 512 and
    # 256 terms with random signs their effect stays under the largest elementary one in the 2-norm
    assert float((y.double() - want).norm() / want.norm()) < 3 * 2.0 ** -4
    got = ctc_amd.expert_layer(x, up, su, down, sd, pick, gate)
    assert bool(((got.double() - want).abs() <= bound).all())


def test_captured_chain_replays_like_the_eager_one(cuda):
    """Quantiser, products (split, skinny, grouped) and the layer in one graph, replayed on new inputs between eager calls."""
    g = gen(61)
    xs = [torch.randn(150, 4096, generator=g).to(BF16).cuda() for _ in range(4)]
    W = (torch.randn(256, 4096, generator=g) * 0.02).cuda()
    qw, sw = ctc_amd.block_quantize(W, "tiles")
    Be, sbe = ref.random_operand(g, (3, 128, 256), "tiles")
    off = offsets_of([40, 0, 110])
    lx, up, su, down, sd, pick, gate = layer_inputs(62, 8, 2, 6, 256, 128)

    def chain(x):
        q, s = ctc_amd.block_quantize(x)
        y = ctc_amd.scaled_contract(q, s, qw, sw)
        one = ctc_amd.scaled_contract(q[:1], s[:1], qw, sw, dtype=F32)
        q2, s2 = ctc_amd.block_quantize(y, transposed=False)
        z = ctc_amd.scaled_grouped_contract(q2, s2, Be, sbe, off)
        w = ctc_amd.expert_layer(y[:8], up, su, down, sd, pick, gate)
        return y, one, z, w

    want = [[v.clone() for v in chain(x)] for x in xs]
    x = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(x)
    for i in (1, 3, 0, 2, 1):
        x.copy_(xs[i])
        graph.replay()
        chain(xs[(i + 1) % 4])  # the program's own work in between
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)


def test_calls_on_several_streams(cuda):
    """Split products and layers that overlap on two streams share no workspace."""
    g = gen(71)
    A, sa = ref.random_operand(g, (2, 150, 16384), "rows")
    B, sb = ref.random_operand(g, (260, 16384), "tiles")
    args = [layer_inputs(72 + i, 8, 2, 6, 256, 128) for i in range(2)]
    want = [(ctc_amd.scaled_contract(A[i], sa[i], B, sb, dtype=F32), ctc_amd.expert_layer(*args[i])) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            got[i].append((ctc_amd.scaled_contract(A[i], sa[i], B, sb, dtype=F32, stream=s),
                           ctc_amd.expert_layer(*args[i], stream=s.cuda_stream)))
    torch.cuda.synchronize()
    for i in range(2):
        for p, y in got[i]:
            assert torch.equal(p, want[i][0]) and torch.equal(y, want[i][1])


def test_python_layer_refuses_before_anything_runs(cuda):
    g = gen(81)
    A, sa = ref.random_operand(g, (40, 256), "rows")
    B, sb = ref.random_operand(g, (30, 256), "tiles")
    off = offsets_of([40])
    for call in (
        lambda: ctc_amd.scaled_contract(A, sa[:, :1], B, sb),
        lambda: ctc_amd.scaled_contract(A, sa.double(), B, sb),
        lambda: ctc_amd.scaled_contract(A, sa, B[:, :128], sb[:, :1]),
        lambda: ctc_amd.scaled_contract(A, sa, B, sb.cpu()),
        lambda: ctc_amd.scaled_contract(A, sa, B, sb, dtype=torch.float64),
        lambda: ctc_amd.scaled_contract(A, sa, B, sb, beta=1.0),
        lambda: ctc_amd.scaled_contract(A, sa, B, sb, out=torch.empty(40, 31, device="cuda")),
        lambda: ctc_amd.scaled_contract(A, sa, B, sb, out=torch.empty(30, 40, device="cuda").t()),
        lambda: ctc_amd.scaled_contract(A.view(torch.uint8), sa, B, sb),
        lambda: ctc_amd.scaled_contract(A.t(), sa, B, sb),
        lambda: ctc_amd.scaled_grouped_contract(A, sa, B[None], sb[None], off.long()),
        lambda: ctc_amd.scaled_grouped_contract(A, sa, B[None], sb[None], offsets_of([20, 20])),
        lambda: ctc_amd.scaled_grouped_contract(A, sa, B[None], sb[None], off, along="columns"),
        lambda: ctc_amd.block_quantize(torch.zeros(4, 256, device="cuda").t()),
        lambda: ctc_amd.block_quantize(torch.zeros(256, device="cuda")),
        lambda: ctc_amd.block_quantize(torch.zeros(4, 256, device="cuda"), out=(A, sa)),
        lambda: ctc_amd.expert_layer(A, A, sa, B, sb, off, off),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ctc_amd.CtcError):
        ctc_amd.scaled_contract(B, sb, A.view(torch.uint8).view(E5M2), sa)
    x, up, su, down, sd, pick, gate = layer_inputs(82, 4, 2, 3, 128, 128)
    with pytest.raises(ctc_amd.CtcError):
        ctc_amd.expert_layer(x.repeat(17, 1), up, su, down, sd, pick.repeat(17, 1), gate.repeat(17, 1))

"""The block-scaled operators in 64 bits, written from their definitions, and how far a kernel in f32 may be off."""
import torch

BLOCK = 128
LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # finfo.eps / 2
F32 = 2.0 ** -24


def cdiv(a, b):
    return -(-a // b)


def spread(scale, rows, cols):
    """Element-wise scales of a rows x cols matrix."""
    s = scale.double()
    if s.shape[-2] != rows:
        s = s.repeat_interleave(BLOCK, -2)[..., :rows, :]
    return s.repeat_interleave(BLOCK, -1)[..., :cols]


def values(q, scale):
    return q.double() * spread(scale, q.shape[-2], q.shape[-1])


def quantize(x, block, dtype):
    """(q, scale), the definition's f32 operations on the CPU: two divisions and one product, each rounded once, and one
    rounding to 8 bits."""
    x = x.float().cpu()
    *lead, r, c = x.shape
    h = 1 if block == "rows" else BLOCK
    p = torch.nn.functional.pad(x, (0, -c % BLOCK, 0, -r % h)).reshape(*lead, cdiv(r, h), h, cdiv(c, BLOCK), BLOCK)
    top = torch.where(p.isfinite(), p.abs(), torch.zeros(())).amax((-3, -1)).clamp_min(2.0 ** -100)
    largest = torch.full_like(top, LARGEST[dtype])
    v = p * (largest / top)[..., :, None, :, None]
    v = v.reshape(*lead, cdiv(r, h) * h, cdiv(c, BLOCK) * BLOCK)[..., :r, :c].contiguous()
    return v.to(dtype), top / largest


def random_operand(g, shape, block, dtype=torch.float8_e4m3fn, pitch=None, lead_offset=0):
    """Random codes over the type's whole finite range (both zeros among them) and positive scales over several octaves;
    rows `pitch` apart, the first one `lead_offset` bytes into its allocation."""
    *lead, r, c = shape
    pitch = c if pitch is None else pitch
    n = 1
    for d in lead:
        n *= d
    raw = torch.randint(0, 256, (lead_offset + n * r * pitch,), generator=g, dtype=torch.int16).to(torch.uint8)
    bad = raw.view(dtype).float().isfinite().logical_not()
    raw[bad] = 0
    # bytes that belong to no element are NaN: a kernel that reads them into a sum shows it
    q = raw[lead_offset:].reshape(*lead, r, pitch)
    if pitch > c:
        q[..., c:] = 0x7F
    raw[:lead_offset] = 0x7F
    rows = r if block == "rows" else cdiv(r, BLOCK)
    scale = torch.exp2(torch.rand(*lead, rows, cdiv(c, BLOCK), generator=g) * 8 - 12)
    dev = raw.cuda()
    q = dev[lead_offset:].reshape(*lead, r, pitch).view(dtype)[..., :c]
    return q, scale.cuda()


def product(A, sa, B, sb, k0=0, k1=None):
    """(C, magnitude) in 64 bits over the contracted range [k0, k1)."""
    a, b = values(A, sa)[..., k0:k1], values(B, sb)[..., k0:k1]
    bt = b.transpose(-1, -2).contiguous()
    return a @ bt, a.abs() @ bt.abs()


def product_bound(want, mag, k, dtype, alpha=1.0, beta=0.0, before=None, fast=False):
    """A sum of n terms in f32 in any order is off by at most n 2^-24 times the sum of their magnitudes; the matrix core
    may truncate instead of rounding, which doubles a step.  Inside a block 128 terms, then an FMA with a rounded product
    of two scales for every block, then alpha, beta and one rounding to the result's type.
    fast: the 8-bit form of the matrix core drops from each of eight neighbouring products what lies below 2^-13 of the
    largest of them, so a group of eight is off by at most 8 * 2^-13 of its largest product, which is at most the sum of the group's
    magnitudes."""
    blocks = cdiv(k, BLOCK)
    steps = 2 * (128 + 2) + blocks + 8  # 8: split chunks and partial sums across waves, alpha, beta
    err = (steps * F32 + (2.0 ** -10 if fast else 0.0)) * abs(alpha) * mag
    if before is not None:
        err = err + 4 * F32 * abs(beta) * before.abs()
    return HALF_STEP[dtype] * (want.abs() + err) + err + 1e-37

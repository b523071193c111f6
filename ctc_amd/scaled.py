"""Block-scaled 8-bit operators: quantiser, products, and a mixture-of-experts layer for a few tokens.

An operand is a pair (q, scale): 8-bit codes (torch.float8_e4m3fn, or float8_e5m2 where an operator takes it) of shape
[rows, columns] and float32 scales, one for every 128 columns of a row ("rows": scale [rows, ceil(columns / 128)]) or for
every 128 x 128 tile ("tiles": scale [ceil(rows / 128), ceil(columns / 128)]).  Products contract the LAST index of both
operands.  Batches and experts add a leading index to both tensors.

Everything goes through the C ABI of libctc_tc.so (include/ctc_tc.h); torch owns memory and streams and computes nothing.
Results and workspaces that a call allocates come from torch's caching allocator on the stream that the call runs on, so
calls on several streams, and calls captured in graphs, never share one.
"""
import contextlib
import ctypes

from . import _lib
from ._lib import BF16, BLOCK_ROWS, BLOCK_TILES, F32, F8E4M3, F8E5M2, GROUPS_CONTRACTED, GROUPS_ROWS, ScaledMatrix, check

BLOCK = 128
_KINDS = {"rows": BLOCK_ROWS, "tiles": BLOCK_TILES}
_types = None


def _torch_types():
    """(torch, {8-bit dtype: code}, {16 / 32-bit dtype: code}); torch is imported on first use, as everywhere in the package."""
    global _types
    if _types is None:
        import torch
        _types = (torch, {torch.float8_e4m3fn: F8E4M3, torch.float8_e5m2: F8E5M2}, {torch.float32: F32, torch.bfloat16: BF16})
    return _types


def _where(device, stream):
    """(context to allocate in, raw stream handle) for a call on `device`."""
    torch = _torch_types()[0]
    if stream is None:
        if torch.cuda.current_device() == device.index:
            return None, torch.cuda.current_stream(device).cuda_stream
        return torch.cuda.device(device), torch.cuda.current_stream(device).cuda_stream
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    if stream.device != device:
        raise ValueError("the stream belongs to %s, the operands to %s" % (stream.device, device))
    return torch.cuda.stream(stream), stream.cuda_stream


def _on_device(name, x, device):
    if not x.is_cuda:
        raise ValueError("%s must live in device memory (got a host tensor)" % name)
    if device is not None and x.device != device:
        raise ValueError("%s is on %s, the other operands on %s" % (name, x.device, device))
    return x.device


def _rows_of(name, x):
    """Leading dimension of x's rows; x has unit stride along them."""
    cols = x.shape[-1]
    if cols > 1 and x.stride(-1) != 1:
        raise ValueError("%s needs unit stride along its last index" % name)
    ld = x.stride(-2) if x.shape[-2] > 1 else cols
    if ld < cols:
        raise ValueError("%s: rows overlap (row stride %d, %d columns)" % (name, ld, cols))
    return ld


def _operand(name, q, scale, device, dims):
    """ctc_tc_scaled_matrix of (q, scale); the block kind is read off the scale's shape."""
    torch, codes, _ = _torch_types()
    code = codes.get(q.dtype)
    if code is None:
        raise ValueError("%s holds %s, not an 8-bit type" % (name, q.dtype))
    if q.dim() not in dims:
        raise ValueError("%s has %d indices" % (name, q.dim()))
    _on_device(name, q, device)
    _on_device(name + "'s scale", scale, q.device)
    if scale.dtype is not torch.float32:
        raise ValueError("%s's scale holds %s, not float32" % (name, scale.dtype))
    rows, cols = q.shape[-2], q.shape[-1]
    tiles = -(-rows // BLOCK)
    lead = tuple(q.shape[:-2])
    shape = tuple(scale.shape)
    blocks = -(-cols // BLOCK)
    if shape == lead + (tiles, blocks):
        block = BLOCK_TILES
    elif shape == lead + (rows, blocks):
        block = BLOCK_ROWS
    else:
        raise ValueError("%s: scale of shape %s fits neither rows %s nor tiles %s" % (name, shape, lead + (rows, blocks), lead + (tiles, blocks)))
    ld = _rows_of(name, q)
    stride = scale.stride()
    batched = q.dim() == 3
    return ScaledMatrix(q.data_ptr(), ld, q.stride(0) if batched else 0, scale.data_ptr(), stride[-2], stride[-1],
                        stride[0] if batched else 0, code, block)


def _result(out, shape, dtype, device, name="out"):
    """(the result, its type code, leading dimension, batch stride); allocated where `out` is None."""
    torch, _, wide = _torch_types()
    if out is None:
        if dtype not in wide:
            raise ValueError("the result is float32 or bfloat16, not %s" % dtype)
        out = torch.empty(shape, dtype=dtype, device=device)
    else:
        if out.dtype not in wide:
            raise ValueError("%s is float32 or bfloat16, not %s" % (name, out.dtype))
        if tuple(out.shape) != tuple(shape):
            raise ValueError("%s has shape %s, the product %s" % (name, tuple(out.shape), tuple(shape)))
        _on_device(name, out, device)
    return out, wide[out.dtype], _rows_of(name, out), out.stride(0) if out.dim() == 3 else 0


def _empty_codes(lead, rows, cols, dtype, device):
    """Codes with rows at multiples of 16 bytes, and group-major scales."""
    torch = _torch_types()[0]
    pitch = -(-cols // 16) * 16
    q = torch.empty(lead + (rows, pitch), dtype=dtype, device=device)
    return q if pitch == cols else q[..., :cols]


def _empty_scale(lead, rows, cols, kind, device):
    torch = _torch_types()[0]
    r = rows if kind == BLOCK_ROWS else -(-rows // BLOCK)
    return torch.empty(lead + (-(-cols // BLOCK), r), dtype=torch.float32, device=device).transpose(-1, -2)


def block_quantize(x, block="rows", dtype=None, transposed=False, out=None, stream=None):
    """8-bit codes and scales of x ([rows, columns] or [batch, rows, columns], float32 or bfloat16, unit column stride).

    block       "rows": one scale for every 128 columns of a row; "tiles": one for every 128 x 128 tile
    dtype       torch.float8_e4m3fn (default) or torch.float8_e5m2
    transposed  False: returns (q, scale); True: (q, scale) of x's transpose, its blocks along the rows of x;
                "both": (q, scale, q_t, scale_t) from one reading of x
    out         the tensors to write instead of new ones, in the order of the result

    scale = top / L and q = round(x * (L / top)) with top the largest finite magnitude of the block, at least 2^-100, and
    L the largest number of the type.  New codes have row pitches of multiples of 16 bytes and new scales keep the index
    of the rows fastest in memory.
    """
    torch, codes, wide = _torch_types()
    if block not in _KINDS:
        raise ValueError("block is 'rows' or 'tiles', not %r" % (block,))
    kind = _KINDS[block]
    if dtype is None:
        dtype = torch.float8_e4m3fn
    if dtype not in codes:
        raise ValueError("dtype is float8_e4m3fn or float8_e5m2, not %s" % dtype)
    if transposed not in (False, True, "both"):
        raise ValueError("transposed is False, True or 'both', not %r" % (transposed,))
    if x.dtype not in wide:
        raise ValueError("x is float32 or bfloat16, not %s" % x.dtype)
    if x.dim() not in (2, 3):
        raise ValueError("x has %d indices" % x.dim())
    device = _on_device("x", x, None)
    ldx = _rows_of("x", x)
    rows, cols = x.shape[-2], x.shape[-1]
    lead = tuple(x.shape[:-2])
    plain, turned = transposed != True, transposed is not False  # noqa: E712
    where, raw = _where(device, stream)
    with where or contextlib.nullcontext():
        if out is None:
            out = ()
            if plain:
                out += (_empty_codes(lead, rows, cols, dtype, device), _empty_scale(lead, rows, cols, kind, device))
            if turned:
                out += (_empty_codes(lead, cols, rows, dtype, device), _empty_scale(lead, cols, rows, kind, device))
        else:
            out = tuple(out)
            if len(out) != 2 * (plain + turned):
                raise ValueError("out has %d tensors, the result %d" % (len(out), 2 * (plain + turned)))
        wanted = ([(rows, cols)] if plain else []) + ([(cols, rows)] if turned else [])
        args = []
        for i, (r, c) in enumerate(wanted):
            q, s = out[2 * i], out[2 * i + 1]
            if q.dtype is not dtype or tuple(q.shape) != lead + (r, c):
                raise ValueError("out[%d] has type %s and shape %s, the result %s and %s" % (2 * i, q.dtype, tuple(q.shape), dtype, lead + (r, c)))
            m = _operand("out[%d]" % (2 * i), q, s, device, (2, 3))
            if m.block != kind and r > 1:
                raise ValueError("out[%d] has the shape of the other block kind" % (2 * i + 1))
            m.block = kind
            args.append(ctypes.byref(m))
        check(_lib.load().ctc_tc_block_quantize(
            x.data_ptr(), rows, cols, ldx, lead[0] if lead else 1, x.stride(0) if lead else 0, wide[x.dtype],
            args[0] if plain else None, args[-1] if turned else None, raw))
    return out


def scaled_contract(A, scale_a, B, scale_b, out=None, dtype=None, alpha=1.0, beta=0.0, stream=None):
    """out[m, n] = alpha * sum_k A[m, k] B[n, k] + beta * out[m, n] of block-scaled operands ([batch, ...] on all or none).

    A is float8_e4m3fn or float8_e5m2, B float8_e4m3fn, either with row or tile scales (read off the scales' shapes).
    The result is `out` (float32 or bfloat16, unit column stride; needed where beta is not 0) or a new tensor of `dtype`
    (bfloat16 by default); sums are float32, rounded once.
    """
    torch = _torch_types()[0]
    device = _on_device("A", A, None)
    a = _operand("A", A, scale_a, device, (2, 3))
    b = _operand("B", B, scale_b, device, (2, 3))
    if A.dim() != B.dim() or A.shape[:-2] != B.shape[:-2] or A.shape[-1] != B.shape[-1]:
        raise ValueError("shapes %s and %s do not contract" % (tuple(A.shape), tuple(B.shape)))
    if out is None and beta != 0:
        raise ValueError("beta needs an `out` to add to")
    L = _lib.load()
    m, k = A.shape[-2], A.shape[-1]
    n = B.shape[-2]
    lead = tuple(A.shape[:-2])
    batch = lead[0] if lead else 1
    where, raw = _where(device, stream)
    with where or contextlib.nullcontext():
        out, code, ldc, stride = _result(out, lead + (m, n), dtype or torch.bfloat16, device)
        room = check(L.ctc_tc_scaled_workspace_bytes(m, n, k, batch))
        ws = torch.empty(room, dtype=torch.uint8, device=device) if room else None
        check(L.ctc_tc_scaled_contract(m, n, k, batch, ctypes.byref(a), ctypes.byref(b), float(alpha), float(beta), out.data_ptr(), ldc,
                                       stride, code, ws.data_ptr() if room else None, room, raw))
    return out


def scaled_grouped_contract(A, scale_a, B, scale_b, offsets, along="rows", out=None, dtype=None, alpha=1.0, beta=0.0, stream=None):
    """Block-scaled products over ragged groups (experts) in one launch; offsets: int32 device tensor of groups + 1 values.

    along="rows"        out[r] = A[r] B[g]^T for the rows r of group g; A [rows, k], B [groups, n, k], out [rows, n].  Rows outside
                        every group are not written.
    along="contracted"  out[g] = sum over the group's range of k of A[m, k] B[n, k]; A [m, k], B [n, k], out [groups, m, n].  The
                        offsets are multiples of 128, or k itself.
    The offsets are read on the device only; see ctc_tc_scaled_grouped_contract for what out-of-range ones do.
    """
    torch = _torch_types()[0]
    if along not in ("rows", "contracted"):
        raise ValueError("along is 'rows' or 'contracted', not %r" % (along,))
    rows = along == "rows"
    device = _on_device("A", A, None)
    a = _operand("A", A, scale_a, device, (2,))
    b = _operand("B", B, scale_b, device, (3,) if rows else (2,))
    if A.shape[-1] != B.shape[-1]:
        raise ValueError("shapes %s and %s do not contract" % (tuple(A.shape), tuple(B.shape)))
    _on_device("offsets", offsets, device)
    if offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 1 or (offsets.shape[0] > 1 and offsets.stride(0) != 1):
        raise ValueError("offsets is a packed int32 vector of groups + 1 values")
    groups = offsets.shape[0] - 1
    if rows and groups != B.shape[0]:
        raise ValueError("%d groups of offsets, %d of B" % (groups, B.shape[0]))
    if out is None and beta != 0:
        raise ValueError("beta needs an `out` to add to")
    m, k = A.shape
    n = B.shape[-2]
    where, raw = _where(device, stream)
    with where or contextlib.nullcontext():
        out, code, ldc, stride = _result(out, (m, n) if rows else (groups, m, n), dtype or torch.bfloat16, device)
        check(_lib.load().ctc_tc_scaled_grouped_contract(
            GROUPS_ROWS if rows else GROUPS_CONTRACTED, groups, offsets.data_ptr(), m, n, k, ctypes.byref(a), ctypes.byref(b), float(alpha),
            float(beta), out.data_ptr(), ldc, stride, code, raw))
    return out


def expert_layer(x, up, scale_up, down, scale_down, pick, gate, out=None, stream=None):
    """y[t] = sum_j gate[t, j] * D_e (silu(G_e x[t]) * (U_e x[t])), e = pick[t, j], for at most 64 tokens.

    x [tokens, hidden] bfloat16; up [experts, 2 inner, hidden] (G over U) and down [experts, hidden, inner] float8_e4m3fn
    with tile scales; pick int32 and gate float32 [tokens, top], top <= 16.  A pick outside the experts contributes nothing.
    Returns y [tokens, hidden] bfloat16 (`out` where given).
    """
    torch = _torch_types()[0]
    device = _on_device("x", x, None)
    if x.dim() != 2 or x.dtype is not torch.bfloat16:
        raise ValueError("x is a bfloat16 matrix, not %s of %d indices" % (x.dtype, x.dim()))
    u = _operand("up", up, scale_up, device, (3,))
    d = _operand("down", down, scale_down, device, (3,))
    tokens, hidden = x.shape
    experts, inner = down.shape[0], down.shape[2]
    if tuple(up.shape) != (experts, 2 * inner, hidden) or down.shape[1] != hidden:
        raise ValueError("shapes of x %s, up %s and down %s do not fit" % (tuple(x.shape), tuple(up.shape), tuple(down.shape)))
    _on_device("pick", pick, device)
    _on_device("gate", gate, device)
    if pick.dim() != 2 or pick.shape[0] != tokens or pick.dtype is not torch.int32 or tuple(gate.shape) != tuple(pick.shape) or gate.dtype is not torch.float32:
        raise ValueError("pick (int32) and gate (float32) are [tokens, top] matrices")
    top = pick.shape[1]
    L = _lib.load()
    where, raw = _where(device, stream)
    with where or contextlib.nullcontext():
        if out is not None and out.dtype is not torch.bfloat16:
            raise ValueError("out is bfloat16, not %s" % out.dtype)
        out, _, ldy, _ = _result(out, (tokens, hidden), torch.bfloat16, device)
        room = check(L.ctc_tc_expert_workspace_bytes(tokens, top, inner))
        ws = torch.empty(max(room, 1), dtype=torch.uint8, device=device)
        check(L.ctc_tc_expert_layer(tokens, top, experts, hidden, inner, x.data_ptr(), _rows_of("x", x), ctypes.byref(u), ctypes.byref(d),
                                    pick.data_ptr(), _rows_of("pick", pick), gate.data_ptr(), _rows_of("gate", gate), out.data_ptr(), ldy,
                                    ws.data_ptr(), max(room, 1), raw))
    return out

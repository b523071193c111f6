"""Block-scaled 8-bit operators: quantiser, products, and a mixture-of-experts layer for a few tokens.

An operand is a pair (q, scale): 8-bit codes (torch.float8_e4m3fn, or float8_e5m2 where an operator takes it) of shape
[rows, columns] and float32 scales, one for every 128 columns of a row ("rows": scale [rows, ceil(columns / 128)]) or for
every 128 x 128 tile ("tiles": scale [ceil(rows / 128), ceil(columns / 128)]).  Products contract the LAST index of both
operands.  Batches and experts add a leading index to both tensors.

Everything goes through the C ABI of libctc_tc.so (include/ctc_tc.h); torch owns memory and streams and computes nothing.
Results and workspaces that a call allocates come from torch's caching allocator on the stream that the call runs on, so
calls on several streams, and calls captured in graphs, never share one.
"""
import ctypes

from . import _lib
from ._lib import BF16, BLOCK_ROWS, BLOCK_TILES, F32, F8E4M3, F8E5M2, GROUPS_CONTRACTED, GROUPS_ROWS, ScaledMatrix, check

BLOCK = 128
_KINDS = {"rows": BLOCK_ROWS, "tiles": BLOCK_TILES}
_byref = ctypes.byref
_state = None


class _State:
    """What every call needs of torch and the library; made on first use (torch is imported nowhere else in the package's top)."""

    def __init__(self):
        import torch
        self.torch = torch
        self.lib = _lib.load()
        self.codes = {torch.float8_e4m3fn: F8E4M3, torch.float8_e5m2: F8E5M2}
        self.wide = {torch.float32: F32, torch.bfloat16: BF16}
        self.f32, self.bf16, self.i32 = torch.float32, torch.bfloat16, torch.int32
        self.empty, self.empty_strided = torch.empty, torch.empty_strided
        # a microsecond and a half faster than the stream object, in calls that take eight
        self.raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
        self.current_device = torch.cuda.current_device


def _get():
    global _state
    if _state is None:
        _state = _State()
    return _state


def _run(st, device, stream, call):
    """call(raw stream handle), with `device` current and allocations made on the stream that the call runs on."""
    if stream is None:
        if st.current_device() == device.index:
            return call(st.raw_stream(device.index))
        with st.torch.cuda.device(device):
            return call(st.raw_stream(device.index))
    cuda = st.torch.cuda
    if isinstance(stream, int):
        stream = cuda.ExternalStream(stream, device=device) if stream else cuda.default_stream(device)
    if stream.device != device:
        raise ValueError("the stream belongs to %s, the operands to %s" % (stream.device, device))
    with cuda.stream(stream):
        return call(stream.cuda_stream)


def _on_device(name, x, device):
    if not x.is_cuda:
        raise ValueError("%s must live in device memory (got a host tensor)" % name)
    if device is not None and x.device != device:
        raise ValueError("%s is on %s, the other operands on %s" % (name, x.device, device))
    return x.device


def _pitch(name, shape, stride):
    """Leading dimension of rows with unit stride along them."""
    cols = shape[-1]
    if cols > 1 and stride[-1] != 1:
        raise ValueError("%s needs unit stride along its last index" % name)
    if shape[-2] <= 1:
        return cols
    if stride[-2] < cols:
        raise ValueError("%s: rows overlap (row stride %d, %d columns)" % (name, stride[-2], cols))
    return stride[-2]


def _operand(st, name, q, scale, device, dims):
    """(ctc_tc_scaled_matrix of (q, scale), shape of q); the block kind is read off the scale's shape."""
    code = st.codes.get(q.dtype)
    if code is None:
        raise ValueError("%s holds %s, not an 8-bit type" % (name, q.dtype))
    shape = tuple(q.shape)
    if len(shape) not in dims:
        raise ValueError("%s has %d indices" % (name, len(shape)))
    if not (q.is_cuda and scale.is_cuda and q.device == device and scale.device == device):
        _on_device(name, q, device)
        _on_device(name + "'s scale", scale, device)
    if scale.dtype is not st.f32:
        raise ValueError("%s's scale holds %s, not float32" % (name, scale.dtype))
    rows, cols = shape[-2:]
    got, blocks = tuple(scale.shape), -(-cols // BLOCK)
    if got == shape[:-2] + (-(-rows // BLOCK), blocks):
        block = BLOCK_TILES
    elif got == shape[:-2] + (rows, blocks):
        block = BLOCK_ROWS
    else:
        raise ValueError("%s: scale of shape %s fits neither the rows nor the tiles of %s" % (name, got, shape))
    stride, s = q.stride(), scale.stride()
    ld = _pitch(name, shape, stride)
    if len(shape) == 3:
        return ScaledMatrix(q.data_ptr(), ld, stride[0], scale.data_ptr(), s[1], s[2], s[0], code, block), shape
    return ScaledMatrix(q.data_ptr(), ld, 0, scale.data_ptr(), s[0], s[1], 0, code, block), shape


def _result(st, out, shape, dtype, device):
    """(the result, its type code, leading dimension, batch stride); allocated where `out` is None."""
    if out is None:
        code = st.wide.get(dtype)
        if code is None:
            raise ValueError("the result is float32 or bfloat16, not %s" % dtype)
        return st.empty(shape, dtype=dtype, device=device), code, shape[-1], shape[-2] * shape[-1]
    code = st.wide.get(out.dtype)
    if code is None:
        raise ValueError("out is float32 or bfloat16, not %s" % out.dtype)
    if tuple(out.shape) != shape:
        raise ValueError("out has shape %s, the result %s" % (tuple(out.shape), shape))
    _on_device("out", out, device)
    stride = out.stride()
    return out, code, _pitch("out", shape, stride), stride[0] if len(shape) == 3 else 0


def _new_codes(st, lead, rows, cols, dtype, code, kind, device):
    """(q, scale, descriptor): rows at multiples of 16 bytes, the index of the rows fastest in the scales."""
    pitch = -(-cols // 16) * 16
    q = st.empty(lead + (rows, pitch), dtype=dtype, device=device)
    if pitch != cols:
        q = q[..., :cols]
    r, b = rows if kind == BLOCK_ROWS else -(-rows // BLOCK), -(-cols // BLOCK)
    scale = st.empty_strided(lead + (b, r)[::-1], (r * b, 1, r) if lead else (1, r), dtype=st.f32, device=device)
    return q, scale, ScaledMatrix(q.data_ptr(), pitch, rows * pitch, scale.data_ptr(), 1, r, r * b, code, kind)


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
    st = _get()
    kind = _KINDS.get(block)
    if kind is None:
        raise ValueError("block is 'rows' or 'tiles', not %r" % (block,))
    if dtype is None:
        dtype = st.torch.float8_e4m3fn
    code = st.codes.get(dtype)
    if code is None:
        raise ValueError("dtype is float8_e4m3fn or float8_e5m2, not %s" % dtype)
    if transposed not in (False, True, "both"):
        raise ValueError("transposed is False, True or 'both', not %r" % (transposed,))
    src = st.wide.get(x.dtype)
    if src is None:
        raise ValueError("x is float32 or bfloat16, not %s" % x.dtype)
    shape = tuple(x.shape)
    if len(shape) not in (2, 3):
        raise ValueError("x has %d indices" % len(shape))
    device = _on_device("x", x, None)
    stride = x.stride()
    ldx = _pitch("x", shape, stride)
    rows, cols = shape[-2:]
    lead = shape[:-2]
    plain, turned = transposed == "both" or not transposed, bool(transposed)
    given = None
    if out is not None:
        given = tuple(out)
        if len(given) != 2 * (plain + turned):
            raise ValueError("out has %d tensors, the result %d" % (len(given), 2 * (plain + turned)))

    def call(raw):
        result, args = (), []
        for wanted, r, c in ((plain, rows, cols), (turned, cols, rows)):
            if not wanted:
                args.append(None)
                continue
            if given is None:
                q, s, m = _new_codes(st, lead, r, c, dtype, code, kind, device)
            else:
                q, s = given[len(result):len(result) + 2]
                m, got = _operand(st, "out[%d]" % len(result), q, s, device, (2, 3))
                if q.dtype is not dtype or got != lead + (r, c):
                    raise ValueError("out[%d] has type %s and shape %s, the result %s and %s" % (len(result), q.dtype, got, dtype, lead + (r, c)))
                if m.block != kind and r > 1:
                    raise ValueError("out[%d] has the shape of the other block kind" % (len(result) + 1))
                m.block = kind
            result += (q, s)
            args.append(_byref(m))
        check(st.lib.ctc_tc_block_quantize(x.data_ptr(), rows, cols, ldx, lead[0] if lead else 1, stride[0] if lead else 0, src, args[0], args[1], raw))
        return result

    return _run(st, device, stream, call)


def scaled_contract(A, scale_a, B, scale_b, out=None, dtype=None, alpha=1.0, beta=0.0, stream=None):
    """out[m, n] = alpha * sum_k A[m, k] B[n, k] + beta * out[m, n] of block-scaled operands ([batch, ...] on all or none).

    A is float8_e4m3fn or float8_e5m2, B float8_e4m3fn, either with row or tile scales (read off the scales' shapes).
    The result is `out` (float32 or bfloat16, unit column stride; needed where beta is not 0) or a new tensor of `dtype`
    (bfloat16 by default), rounded once.  A float32 result takes float32 sums throughout; ctc_tc_scaled_contract says what a
    large bfloat16 one takes.
    """
    st = _get()
    device = _on_device("A", A, None)
    a, sa = _operand(st, "A", A, scale_a, device, (2, 3))
    b, sb = _operand(st, "B", B, scale_b, device, (2, 3))
    if sa[:-2] != sb[:-2] or sa[-1] != sb[-1]:
        raise ValueError("shapes %s and %s do not contract" % (sa, sb))
    if out is None and beta != 0:
        raise ValueError("beta needs an `out` to add to")
    m, k = sa[-2:]
    n = sb[-2]
    lead = sa[:-2]
    batch = lead[0] if lead else 1

    def call(raw):
        c, code, ldc, stride = _result(st, out, lead + (m, n), dtype or st.bf16, device)
        # (32: products of so few rows never split; a negative answer: the operator refuses the sizes too, with its own words)
        room = max(st.lib.ctc_tc_scaled_workspace_bytes(m, n, k, batch), 0) if m > 32 else 0
        ws = st.empty(room, dtype=st.torch.uint8, device=device) if room else None
        check(st.lib.ctc_tc_scaled_contract(m, n, k, batch, _byref(a), _byref(b), float(alpha), float(beta), c.data_ptr(), ldc, stride, code,
                                            ws.data_ptr() if room else None, room, raw))
        return c

    return _run(st, device, stream, call)


def scaled_grouped_contract(A, scale_a, B, scale_b, offsets, along="rows", out=None, dtype=None, alpha=1.0, beta=0.0, stream=None):
    """Block-scaled products over ragged groups (experts) in one launch; offsets: int32 device tensor of groups + 1 values.

    along="rows"        out[r] = A[r] B[g]^T for the rows r of group g; A [rows, k], B [groups, n, k], out [rows, n].  Rows outside
                        every group are not written.
    along="contracted"  out[g] = sum over the group's range of k of A[m, k] B[n, k]; A [m, k], B [n, k], out [groups, m, n].  The
                        offsets are multiples of 128, or k itself.
    The offsets are read on the device only; see ctc_tc_scaled_grouped_contract for what out-of-range ones do.
    """
    st = _get()
    if along not in ("rows", "contracted"):
        raise ValueError("along is 'rows' or 'contracted', not %r" % (along,))
    rows = along == "rows"
    device = _on_device("A", A, None)
    a, sa = _operand(st, "A", A, scale_a, device, (2,))
    b, sb = _operand(st, "B", B, scale_b, device, (3,) if rows else (2,))
    if sa[-1] != sb[-1]:
        raise ValueError("shapes %s and %s do not contract" % (sa, sb))
    _on_device("offsets", offsets, device)
    if offsets.dtype is not st.i32 or offsets.dim() != 1 or offsets.shape[0] < 1 or (offsets.shape[0] > 1 and offsets.stride(0) != 1):
        raise ValueError("offsets is a packed int32 vector of groups + 1 values")
    groups = offsets.shape[0] - 1
    if rows and groups != sb[0]:
        raise ValueError("%d groups of offsets, %d of B" % (groups, sb[0]))
    if out is None and beta != 0:
        raise ValueError("beta needs an `out` to add to")
    m, k = sa
    n = sb[-2]

    def call(raw):
        c, code, ldc, stride = _result(st, out, (m, n) if rows else (groups, m, n), dtype or st.bf16, device)
        check(st.lib.ctc_tc_scaled_grouped_contract(GROUPS_ROWS if rows else GROUPS_CONTRACTED, groups, offsets.data_ptr(), m, n, k, _byref(a),
                                                    _byref(b), float(alpha), float(beta), c.data_ptr(), ldc, stride, code, raw))
        return c

    return _run(st, device, stream, call)


def expert_layer(x, up, scale_up, down, scale_down, pick, gate, out=None, stream=None):
    """y[t] = sum_j gate[t, j] * D_e (silu(G_e x[t]) * (U_e x[t])), e = pick[t, j], for at most 64 tokens.

    x [tokens, hidden] bfloat16; up [experts, 2 inner, hidden] (G over U) and down [experts, hidden, inner] float8_e4m3fn
    with tile scales; pick int32 and gate float32 [tokens, top], top <= 16.  A pick outside the experts contributes nothing.
    Returns y [tokens, hidden] bfloat16 (`out` where given).
    """
    st = _get()
    device = _on_device("x", x, None)
    shape = tuple(x.shape)
    if len(shape) != 2 or x.dtype is not st.bf16:
        raise ValueError("x is a bfloat16 matrix, not %s of %d indices" % (x.dtype, len(shape)))
    u, su = _operand(st, "up", up, scale_up, device, (3,))
    d, sd = _operand(st, "down", down, scale_down, device, (3,))
    tokens, hidden = shape
    experts, inner = sd[0], sd[2]
    if su != (experts, 2 * inner, hidden) or sd[1] != hidden:
        raise ValueError("shapes of x %s, up %s and down %s do not fit" % (shape, su, sd))
    _on_device("pick", pick, device)
    _on_device("gate", gate, device)
    picks = tuple(pick.shape)
    if len(picks) != 2 or picks[0] != tokens or pick.dtype is not st.i32 or tuple(gate.shape) != picks or gate.dtype is not st.f32:
        raise ValueError("pick (int32) and gate (float32) are [tokens, top] matrices")
    if out is not None and out.dtype is not st.bf16:
        raise ValueError("out is bfloat16, not %s" % out.dtype)
    top = picks[1]
    ldx, ld_pick, ld_gate = _pitch("x", shape, x.stride()), _pitch("pick", picks, pick.stride()), _pitch("gate", picks, gate.stride())

    def call(raw):
        y, _, ldy, _ = _result(st, out, shape, st.bf16, device)
        room = max(st.lib.ctc_tc_expert_workspace_bytes(tokens, top, inner), 1)  # (negative: as in scaled_contract)
        ws = st.empty(room, dtype=st.torch.uint8, device=device)
        check(st.lib.ctc_tc_expert_layer(tokens, top, experts, hidden, inner, x.data_ptr(), ldx, _byref(u), _byref(d), pick.data_ptr(), ld_pick,
                                         gate.data_ptr(), ld_gate, y.data_ptr(), ldy, ws.data_ptr(), room, raw))
        return y

    return _run(st, device, stream, call)

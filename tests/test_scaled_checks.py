"""Refusals of the block-scaled operators: nothing is launched, so no GPU is needed."""
import ctypes

import pytest
import torch

import ctc_amd
from ctc_amd import _lib

EINVAL, EUNSUPPORTED, EALIGN = -1, -5, -6
ADDR = 1 << 20  # never dereferenced: every call below is refused, or has nothing to do


def matrix(q=ADDR, ld=256, batch=0, scale=ADDR, dtype=_lib.F8E4M3, block=_lib.BLOCK_ROWS, s_row=1, s_blk=64, s_batch=0):
    return _lib.ScaledMatrix(q, ld, batch, scale, s_row, s_blk, s_batch, dtype, block)


def ref(m):
    return None if m is None else ctypes.byref(m)


def quantize(rows=8, cols=256, ldx=256, batch=1, stride=0, src=_lib.BF16, x=ADDR, out=matrix(), out_t=None):
    return _lib.load().ctc_tc_block_quantize(x, rows, cols, ldx, batch, stride, src, ref(out), ref(out_t), None)


def product(m=64, n=64, k=256, batch=1, a=matrix(), b=matrix(), C=ADDR, ldc=64, stride=0, dtype=_lib.BF16, ws=None, room=0):
    return _lib.load().ctc_tc_scaled_contract(m, n, k, batch, ref(a), ref(b), 1.0, 0.0, C, ldc, stride, dtype, ws, room, None)


def grouped(along=_lib.GROUPS_ROWS, groups=4, offsets=ADDR, m=64, n=64, k=256, a=matrix(), b=matrix(), C=ADDR, ldc=64, stride=64 * 64,
            dtype=_lib.BF16):
    return _lib.load().ctc_tc_scaled_grouped_contract(along, groups, offsets, m, n, k, ref(a), ref(b), 1.0, 0.0, C, ldc, stride, dtype, None)


TILES = matrix(block=_lib.BLOCK_TILES)


def experts(tokens=2, top=2, experts=8, hidden=256, inner=256, x=ADDR, ldx=256, up=TILES, down=TILES, pick=ADDR, gate=ADDR, y=ADDR, ldy=256,
            ws=ADDR, room=1 << 20, ld=2):
    return _lib.load().ctc_tc_expert_layer(tokens, top, experts, hidden, inner, x, ldx, ref(up), ref(down), pick, ld, gate, ld, y, ldy, ws,
                                           room, None)


@pytest.mark.parametrize("kw, code", [
    (dict(rows=-1), EINVAL), (dict(cols=-1), EINVAL), (dict(batch=-1), EINVAL), (dict(src=_lib.F64), EUNSUPPORTED), (dict(src=7), EUNSUPPORTED),
    (dict(out=None), EINVAL), (dict(x=None), EINVAL), (dict(ldx=255), EINVAL), (dict(x=ADDR + 1), EALIGN), (dict(src=_lib.F32, x=ADDR + 2), EALIGN),
    (dict(out=matrix(q=None)), EINVAL), (dict(out=matrix(scale=None)), EINVAL), (dict(out=matrix(scale=ADDR + 2)), EALIGN),
    (dict(out=matrix(ld=255)), EINVAL), (dict(out=matrix(dtype=_lib.BF16)), EINVAL), (dict(out=matrix(block=2)), EINVAL),
    (dict(out=matrix(s_row=-1)), EINVAL), (dict(out_t=matrix(ld=7)), EINVAL), (dict(out_t=matrix(dtype=_lib.F8E5M2)), EINVAL),
    (dict(out_t=TILES), EINVAL), (dict(batch=1 << 17, out=matrix(batch=1 << 20, s_batch=1 << 20)), EUNSUPPORTED), (dict(rows=1 << 31), EINVAL), (dict(stride=-1), EINVAL),
    # results that would be written twice: scales of all rows, of both blocks, of both matrices, codes of both matrices
    (dict(out=matrix(s_row=0)), EINVAL), (dict(out=matrix(s_blk=4)), EINVAL), (dict(batch=2, out=matrix(batch=8 * 256)), EINVAL),
    (dict(batch=2, out=matrix(s_batch=128)), EINVAL), (dict(out=matrix(ld=1 << 50)), EUNSUPPORTED), (dict(ldx=1 << 50), EUNSUPPORTED),
])
def test_quantizer_refuses(kw, code):
    assert quantize(**kw) == code
    assert b"block_quantize" in _lib.load().ctc_tc_last_error()


@pytest.mark.parametrize("kw, code", [
    (dict(m=-1), EINVAL), (dict(k=-1), EINVAL), (dict(m=1 << 31), EUNSUPPORTED), (dict(batch=1 << 16), EUNSUPPORTED), (dict(a=None), EINVAL),
    (dict(a=matrix(dtype=_lib.BF16)), EINVAL), (dict(b=matrix(dtype=_lib.F8E5M2)), EUNSUPPORTED), (dict(a=matrix(ld=255)), EINVAL),
    (dict(b=matrix(q=None)), EINVAL), (dict(b=matrix(scale=ADDR + 1)), EALIGN), (dict(C=None), EINVAL), (dict(ldc=63), EINVAL),
    (dict(dtype=_lib.F64), EUNSUPPORTED), (dict(dtype=_lib.F8E4M3), EUNSUPPORTED), (dict(C=ADDR + 1), EALIGN), (dict(dtype=_lib.F32, C=ADDR + 2), EALIGN),
    (dict(batch=2, stride=64), EINVAL), (dict(ws=ADDR + 8, room=64), EALIGN), (dict(room=-1), EINVAL), (dict(a=matrix(ld=1 << 50)), EUNSUPPORTED),
    (dict(ldc=1 << 50), EUNSUPPORTED), (dict(batch=2, stride=-64 * 64), EINVAL),
    # more tiles than a launch takes, and than 64 bits count
    (dict(m=1 << 23, n=1 << 23, ldc=1 << 23, b=matrix(s_blk=1 << 23), a=matrix(s_blk=1 << 23)), EUNSUPPORTED),
    (dict(m=1 << 30, n=1 << 30, batch=65535, ldc=1 << 30, a=matrix(ld=256), b=matrix(ld=256), stride=1 << 60), EUNSUPPORTED),
])
def test_product_refuses(kw, code):
    assert product(**kw) == code
    assert b"scaled_contract" in _lib.load().ctc_tc_last_error()


@pytest.mark.parametrize("kw, code", [
    (dict(along=2), EINVAL), (dict(groups=-1), EINVAL), (dict(offsets=None), EINVAL), (dict(offsets=ADDR + 2), EALIGN), (dict(groups=1 << 16), EUNSUPPORTED),
    (dict(along=_lib.GROUPS_CONTRACTED, stride=64), EINVAL), (dict(b=matrix(dtype=_lib.F8E5M2)), EUNSUPPORTED), (dict(ldc=1), EINVAL), (dict(n=-1), EINVAL),
])
def test_grouped_product_refuses(kw, code):
    assert grouped(**kw) == code
    assert b"scaled_grouped_contract" in _lib.load().ctc_tc_last_error()


@pytest.mark.parametrize("kw, code", [
    (dict(tokens=65), EUNSUPPORTED), (dict(top=17, ld=17), EUNSUPPORTED), (dict(experts=4097), EUNSUPPORTED), (dict(tokens=-1), EINVAL),
    (dict(top=0), EINVAL), (dict(inner=0), EINVAL), (dict(up=matrix()), EUNSUPPORTED), (dict(down=matrix(dtype=_lib.F8E5M2, block=_lib.BLOCK_TILES)), EUNSUPPORTED),
    (dict(x=None), EINVAL), (dict(gate=ADDR + 2), EALIGN), (dict(y=ADDR + 1), EALIGN), (dict(ldx=255), EINVAL), (dict(ld=1), EINVAL),
    (dict(ws=None), EINVAL), (dict(room=2 * 2 * 256 * 2 - 1), EINVAL), (dict(ws=ADDR + 4), EALIGN),
    (dict(ldx=1 << 60), EUNSUPPORTED), (dict(ldy=1 << 50), EUNSUPPORTED), (dict(ld=1 << 62), EUNSUPPORTED),
])
def test_expert_layer_refuses(kw, code):
    assert experts(**kw) == code
    assert b"expert_layer" in _lib.load().ctc_tc_last_error()


def test_quantizer_takes_every_order_of_a_results_indexes():
    """[rows, batch, columns] in memory, scales with the batch fastest: nothing overlaps (no rows, so nothing is launched)."""
    L = _lib.load()
    m = matrix(ld=3 * 256, batch=256, s_row=3, s_blk=3 * 8, s_batch=1)
    assert L.ctc_tc_block_quantize(None, 8, 256, 256, 3, 8 * 256, _lib.BF16, ref(m), None, None) == EINVAL
    assert b"input is null" in L.ctc_tc_last_error()
    assert quantize(batch=3, stride=8 * 256, x=None, out=m) == EINVAL


def test_kernels_that_set_m0_from_assembly_have_no_other_m0_user(tmp_path):
    """The block-scaled products' LDS-DMA transfers overwrite M0 in inline assembly, which cannot be declared: in their code
    every instruction that names M0 must be the move in front of a transfer, and every transfer have one, a wait state apart."""
    import os
    import re
    import shutil
    import subprocess
    objdump = "/opt/rocm/lib/llvm/bin/llvm-objdump"
    if not os.path.exists(objdump):
        pytest.skip("llvm-objdump is not installed")
    lib = tmp_path / "libctc_tc.so"
    shutil.copy(_lib.LIB_PATH, lib)
    subprocess.run([objdump, "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp_path)
    name, last, before, kernels = None, "", "", {}
    for obj in (p for p in tmp_path.iterdir() if "amdgcn" in p.name and p.stat().st_size > 0):
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", str(obj)], check=True, capture_output=True, text=True).stdout
        if "scaled_gemm_kernel" not in text:
            continue
        for line in text.splitlines():
            m = re.match(r"^[0-9a-f]+ <(\S+)>:", line)
            if m:
                name = m.group(1) if "scaled_gemm_kernel" in m.group(1) else None
                continue
            inst = re.sub(r"\s*//.*$", "", line).strip()
            if name is None or not inst:
                continue
            assert not re.match(r"(v_movrel|s_movrel|s_sendmsg|v_interp|ds_gws|v_pk_(add|mul|fma)_f32)", inst), (name, inst)
            if inst.startswith("global_load_lds"):
                kernels[name] = kernels.get(name, 0) + 1
                assert re.match(r"s_mov_b32 m0, s\d+$", before) and last == "s_nop 0", (name, before, last, inst)
            else:
                assert not re.match(r"s_mov_b32 m0", before), (name, before, last, inst)
                assert "m0" not in inst or re.match(r"s_mov_b32 m0, s\d+$", inst), (name, inst)
            before, last = last, inst
    assert len(kernels) == 24, kernels  # two types of A, two of scales: two forms of the large tile, two sums and two depths on the small one


def test_nothing_to_do_succeeds_without_a_device():
    assert quantize(rows=0, out=matrix(q=None, scale=None)) == 0
    assert quantize(batch=0) == 0
    assert product(m=0, C=None) == 0 and product(n=0) == 0 and product(batch=0) == 0
    assert grouped(groups=0) == 0 and grouped(m=0) == 0
    assert experts(tokens=0) == 0


def test_workspace_queries():
    L = _lib.load()
    assert L.ctc_tc_scaled_workspace_bytes(4096, 4096, 4096, 1) == 0
    assert L.ctc_tc_scaled_workspace_bytes(0, 4096, 4096, 1) == 0
    few = L.ctc_tc_scaled_workspace_bytes(128, 256, 16384, 1)
    assert few > 0 and few % (4 * 128 * 256) == 0
    assert L.ctc_tc_scaled_workspace_bytes(-1, 1, 1, 1) == EINVAL
    assert L.ctc_tc_expert_workspace_bytes(3, 2, 100) == 3 * 2 * 100 * 2
    assert L.ctc_tc_expert_workspace_bytes(65, 2, 100) == EINVAL


def test_eight_bit_types_stay_out_of_plans():
    for dtype in (_lib.F8E4M3, _lib.F8E5M2):
        h = ctypes.c_void_p()
        ext = (ctypes.c_int64 * 3)(4, 4, 4)
        assert _lib.load().ctc_tc_plan_create(b"ak,kb->ab", 3, b"abk", ext, None, None, None, dtype, ctypes.byref(h)) < 0


def test_python_layer_refuses_host_tensors_and_wrong_types():
    q = torch.zeros(4, 256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones(4, 2)
    with pytest.raises(ValueError, match="host tensor"):
        ctc_amd.scaled_contract(q, s, q, s)
    with pytest.raises(ValueError, match="host tensor"):
        ctc_amd.block_quantize(torch.zeros(4, 4))
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ctc_amd.block_quantize(torch.zeros(4, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="'rows' or 'tiles'"):
        ctc_amd.block_quantize(torch.zeros(4, 4), "columns")
    with pytest.raises(ValueError, match="transposed"):
        ctc_amd.block_quantize(torch.zeros(4, 4), transposed="yes")
    with pytest.raises(ValueError, match="host tensor"):
        ctc_amd.scaled_grouped_contract(q, s, q[None], s[None], torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="host tensor"):
        ctc_amd.expert_layer(torch.zeros(2, 256, dtype=torch.bfloat16), q[None], s[None], q[None], s[None], None, None)

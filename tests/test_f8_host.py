"""What the 8-bit operators refuse, through the C-ABI and the Python wrappers
(no GPU: every call is rejected before a launch)."""

import pytest
import torch

from tjkernels import _lib, ops
from tjkernels._lib import BF16, E4M3, EINVAL, EUNSUPPORTED, F16, F32, TjkError

FAKE = 1 << 20  # a pointer that is never followed


def _norm(**kw):
    a = dict(res=FAKE, res_dtype=F32, ld_res=256, delta=FAKE, delta_dtype=BF16, ld_delta=256, res_out=FAKE + 4096,
             res_out_dtype=F32, ld_res_out=256, out=FAKE, out_dtype=E4M3, ld_out=256, scales=FAKE, ld_scales=2, gamma=FAKE,
             rows=4, n=256, eps=1e-5, stream=None)
    a.update(kw)
    return _lib.load().tjk_add_rmsnorm(*a.values())


def _quant(**kw):
    a = dict(x=FAKE, x_dtype=BF16, ld_x=256, q=FAKE, ld_q=256, scales=FAKE, ld_scales=2, rows=4, n=256, block_rows=1,
             stream=None)
    a.update(kw)
    return _lib.load().tjk_quantize_f8(*a.values())


def _gemm(**kw):
    a = dict(a=FAKE, lda=256, a_scales=FAKE, ld_as=2, w=FAKE, ldw=256, w_scales=FAKE, ld_ws=2, bias=FAKE, c=FAKE,
             out_dtype=BF16, ldc=128, c_scales=None, ld_cs=0, m=4, n=128, k=256, epilogue=0, plan=-1, stream=None)
    a.update(kw)
    return _lib.load().tjk_gemm_f8(*a.values())


def _said():
    return _lib.load().tjk_last_error_string().decode()


@pytest.mark.parametrize("kw,status,word", [
    (dict(rows=-1), EINVAL, "shape"), (dict(n=0), EINVAL, "shape"), (dict(n=252), EUNSUPPORTED, "multiple of 8"),
    (dict(n=32776), EUNSUPPORTED, "32768"), (dict(res=None), EINVAL, "null"), (dict(out=None), EINVAL, "null"),
    (dict(gamma=None), EINVAL, "null"), (dict(scales=None), EINVAL, "null"),
    (dict(res_dtype=E4M3), EINVAL, "dtype"), (dict(delta_dtype=9), EINVAL, "dtype"),
    (dict(res_out_dtype=E4M3), EINVAL, "dtype"), (dict(out_dtype=4), EINVAL, "dtype"),
    (dict(ld_res=248), EINVAL, "leading"), (dict(ld_out=255), EINVAL, "leading"), (dict(ld_delta=0), EINVAL, "leading"),
    (dict(ld_scales=1), EINVAL, "leading"), (dict(ld_res=260), EUNSUPPORTED, "multiples of 8"),
    (dict(ld_delta=257), EUNSUPPORTED, "multiples of 8"), (dict(res=FAKE + 8), EUNSUPPORTED, "misaligned"),
    (dict(out=FAKE + 4), EUNSUPPORTED, "misaligned"), (dict(scales=FAKE + 2), EUNSUPPORTED, "misaligned"),
    (dict(gamma=FAKE + 4), EUNSUPPORTED, "misaligned"), (dict(res_out=FAKE + 8), EUNSUPPORTED, "misaligned"),
    (dict(res_out=FAKE, res_out_dtype=F16, delta=None), EINVAL, "alias"),
    (dict(res_out=FAKE, ld_res_out=264, delta=None), EINVAL, "alias"),
    (dict(res=FAKE + 64, res_out=FAKE), EINVAL, "alias"),  # fp32 into a bf16 delta
    (dict(rows=1 << 31), EUNSUPPORTED, "int32"),
])
def test_norm_refusals(kw, status, word):
    assert _norm(**kw) == status and word in _said()


@pytest.mark.parametrize("kw,status,word", [
    (dict(rows=-1), EINVAL, "shape"), (dict(n=-8), EINVAL, "shape"), (dict(block_rows=64), EINVAL, "block_rows"),
    (dict(x_dtype=E4M3), EINVAL, "dtype"), (dict(n=100), EUNSUPPORTED, "multiple of 8"),
    (dict(n=(1 << 20) + 8), EUNSUPPORTED, "2^20"), (dict(x=None), EINVAL, "null"), (dict(q=None), EINVAL, "null"),
    (dict(scales=None), EINVAL, "null"), (dict(ld_x=200), EINVAL, "leading"), (dict(ld_q=200), EINVAL, "leading"),
    (dict(ld_scales=1), EINVAL, "leading"), (dict(ld_x=260), EUNSUPPORTED, "multiples of 8"),
    (dict(x=FAKE + 8), EUNSUPPORTED, "misaligned"), (dict(q=FAKE + 4), EUNSUPPORTED, "misaligned"),
    (dict(rows=1 << 40), EUNSUPPORTED, "too many"), (dict(rows=1 << 40, block_rows=128), EUNSUPPORTED, "too many"),
])
def test_quantize_refusals(kw, status, word):
    assert _quant(**kw) == status and word in _said()


@pytest.mark.parametrize("kw,status,word", [
    (dict(m=-1), EINVAL, "negative"), (dict(k=-16), EINVAL, "negative"), (dict(epilogue=2), EINVAL, "epilogue"),
    (dict(epilogue=-1), EINVAL, "epilogue"), (dict(out_dtype=F32), EINVAL, "dtype"), (dict(out_dtype=7), EINVAL, "dtype"),
    (dict(plan=-2), EINVAL, "plan"), (dict(plan=1000), EINVAL, "plan"), (dict(a=None), EINVAL, "null"),
    (dict(w_scales=None), EINVAL, "null"), (dict(out_dtype=E4M3), EINVAL, "null"), (dict(c=None), EINVAL, "null"),
    (dict(k=248), EUNSUPPORTED, "multiple of 16"), (dict(n=126), EUNSUPPORTED, "multiple of 4"),
    (dict(lda=240), EINVAL, "leading"), (dict(ldw=0), EINVAL, "leading"), (dict(ldc=124), EINVAL, "leading"),
    (dict(ld_as=1), EINVAL, "leading"), (dict(ld_ws=1), EINVAL, "leading"),
    (dict(out_dtype=E4M3, c_scales=FAKE, n=256, ldc=256, ld_cs=1), EINVAL, "leading"),
    (dict(lda=264), EUNSUPPORTED, "multiples of 16"), (dict(ldc=130), EUNSUPPORTED, "multiple of 4"),
    (dict(lda=1 << 23), EUNSUPPORTED, "too large"), (dict(ld_as=1 << 21), EUNSUPPORTED, "too large"),
    (dict(a=FAKE + 8), EUNSUPPORTED, "misaligned"), (dict(c=FAKE + 4), EUNSUPPORTED, "misaligned"),
    (dict(bias=FAKE + 2), EUNSUPPORTED, "misaligned"), (dict(a_scales=FAKE + 1), EUNSUPPORTED, "misaligned"),
    (dict(m=1 << 31), EUNSUPPORTED, "int32"),
])
def test_gemm_refusals(kw, status, word):
    assert _gemm(**kw) == status and word in _said()


def test_nothing_to_do_is_no_error():
    assert _norm(rows=0, res=None) == 0
    assert _quant(rows=0, x=None) == 0
    assert _gemm(m=0, a=None) == 0
    assert _gemm(n=0, w=None, ldc=0) == 0


def test_wrappers_take_device_tensors_only():
    x = torch.zeros(4, 128)
    q, s = torch.zeros(4, 128, dtype=ops.F8), torch.zeros(4, 1)
    with pytest.raises(TjkError, match="device tensors"):
        ops.quantize_f8(x, q, s)
    with pytest.raises(TjkError, match="device tensors"):
        ops.add_rmsnorm(x, None, torch.ones(128), 1e-5, q, scales=s)
    with pytest.raises(TjkError, match="device tensors"):
        ops.gemm_f8(q, s, q, s, None, torch.zeros(4, 4, dtype=torch.bfloat16))


def test_scale_layouts():
    """Scales: fp32, enough rows and blocks, unit column stride, no row
    repeated by a zero stride; one row or one block may have any stride.  (What
    is well formed is refused last, for its device.)"""
    def call(s, rows, cols):
        x, q = torch.zeros(rows, cols), torch.zeros(rows, cols, dtype=ops.F8)
        ops.quantize_f8(x, q, s)

    for s, rows, cols in ((torch.zeros(4, 3), 4, 260), (torch.zeros(4, 8)[:, :3], 4, 260), (torch.zeros(5, 8), 4, 260),
                          (torch.zeros(1, 3).t().contiguous().t(), 1, 260), (torch.zeros(4, 8)[:, 2:3], 4, 128)):
        with pytest.raises(TjkError, match="device tensors"):
            call(s, rows, cols)
    for bad in (torch.zeros(4, 2), torch.zeros(3, 3), torch.zeros(4, 3, dtype=torch.float64),
                torch.zeros(3, 4).t(), torch.zeros(1, 3).expand(4, 3), torch.zeros(12)):
        with pytest.raises(TjkError, match="float32"):
            call(bad, 4, 260)


def _bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _e4m3(*shape):
    return torch.zeros(*shape, dtype=ops.F8)


@pytest.mark.parametrize("kw,word", [
    (dict(res=torch.zeros(4, 256).t()), "row-major"), (dict(res=torch.zeros(256)), "row-major"),
    (dict(res=torch.zeros(4, 256, dtype=torch.float64)), "dtype"), (dict(res=[1.0]), "must be a tensor"),
    (dict(res=None), "must be a tensor"), (dict(delta=_bf16(3, 256)), "delta must be"),
    (dict(delta=_bf16(4, 264)), "delta must be"), (dict(delta=torch.zeros(4, 256, dtype=torch.int32)), "dtype"),
    (dict(out=_bf16(4, 248), scales=None), "out must be"), (dict(res_out=torch.zeros(2, 256)), "res_out must be"),
    (dict(gamma=torch.ones(255)), "gamma"), (dict(gamma=_bf16(256)), "gamma"), (dict(gamma=torch.ones(1, 256)), "gamma"),
    (dict(gamma=torch.ones(512)[::2]), "gamma"), (dict(scales=None), "float32"), (dict(scales=torch.zeros(4, 1)), "float32"),
    (dict(out=_bf16(4, 256)), "belong to"), (dict(), "device tensors"),
])
def test_norm_wrapper_refusals(kw, word):
    a = dict(res=torch.zeros(4, 256), delta=_bf16(4, 256), gamma=torch.ones(256), eps=1e-5, out=_e4m3(4, 256),
             res_out=torch.zeros(4, 256), scales=torch.zeros(4, 2))
    a.update(kw)
    with pytest.raises(TjkError, match=word):
        ops.add_rmsnorm(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(out=_bf16(130, 256)), "out must be"), (dict(out=_e4m3(129, 256)), "out must be"),
    (dict(out=_e4m3(130, 264)), "out must be"), (dict(block_rows=64), "block_rows"), (dict(block_rows=1 << 40), "range"),
    (dict(scales=None), "must be a tensor"), (dict(scales=torch.zeros(1, 2)), "float32"),
    (dict(x=torch.zeros(130, 256, dtype=torch.int8)), "dtype"), (dict(x=torch.zeros(256, 130).t()), "row-major"),
    (dict(), "device tensors"),
])
def test_quantize_wrapper_refusals(kw, word):
    a = dict(x=torch.zeros(130, 256), out=_e4m3(130, 256), scales=torch.zeros(2, 2), block_rows=128)
    a.update(kw)
    with pytest.raises(TjkError, match=word):
        ops.quantize_f8(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(a=_bf16(4, 256)), "must be float8"), (dict(w=_bf16(132, 256)), "must be float8"),
    (dict(w=_e4m3(132, 240)), "mismatch"), (dict(out=_bf16(5, 132)), "mismatch"), (dict(out=_bf16(4, 128)), "mismatch"),
    (dict(out=torch.zeros(4, 132)), "out must be"), (dict(out=_e4m3(4, 132), bias=torch.zeros(132)), "out_scales must be"),
    (dict(out_scales=torch.zeros(4, 2)), "belong to"), (dict(a_scales=torch.zeros(3, 2)), "a_scales"),
    (dict(w_scales=torch.zeros(1, 2)), "w_scales"), (dict(w_scales=torch.zeros(2, 1)), "w_scales"),
    (dict(bias=torch.zeros(132)), "bias"), (dict(bias=_bf16(131)), "bias"), (dict(bias=_bf16(264)[::2]), "bias"),
    (dict(out=_e4m3(4, 132), out_scales=torch.zeros(4, 2)), "bias"), (dict(a=_e4m3(256, 4).t()), "row-major"),
    (dict(plan=1 << 32), "range"), (dict(epilogue=-(1 << 40)), "range"), (dict(bias=None), "device tensors"),
])
def test_gemm_wrapper_refusals(kw, word):
    a = dict(a=_e4m3(4, 256), a_scales=torch.zeros(4, 2), w=_e4m3(132, 256), w_scales=torch.zeros(2, 2), bias=_bf16(132),
             out=_bf16(4, 132))
    a.update(kw)
    with pytest.raises(TjkError, match=word):
        ops.gemm_f8(**a)


def test_wrapper_argument_types():
    a = (torch.zeros(4, 256), None, torch.ones(256), "eps", _bf16(4, 256))
    with pytest.raises(TypeError):
        ops.add_rmsnorm(*a)
    with pytest.raises(TypeError):
        ops.quantize_f8(torch.zeros(4, 256), _e4m3(4, 256), torch.zeros(4, 2), block_rows="1")


def test_every_tile_is_some_shapes_choice():
    """The rule reaches every tile of either list (the second is of e4m3
    outputs), with K groups only where there are few tiles."""
    lib = _lib.load()
    assert lib.tjk_gemm_f8_plan_count() == 9
    shapes = [(m, n, k) for m in (1, 8, 64, 128, 256, 512, 1024, 2443, 5430, 8192, 16384)
              for n in (128, 512, 1024, 2600, 4096, 8192) for k in (128, 512, 1024, 2048, 4096, 8192)]
    for out in (BF16, E4M3):
        got = {lib.tjk_gemm_f8_default_plan(m, n, k, out, e) for m, n, k in shapes for e in (0, 1)}
        assert got == (set(range(9)) if out == BF16 else set(range(3)))
    assert lib.tjk_gemm_f8_default_plan(8192, 8192, 8192, BF16, 0) == 0
    assert lib.tjk_gemm_f8_default_plan(8, 8192, 2048, BF16, 0) == 7
    for bad in ((0, 8, 16, BF16, 0), (8, 8, -1, BF16, 0), (8, 8, 16, F32, 0), (8, 8, 16, BF16, 2)):
        assert lib.tjk_gemm_f8_default_plan(*bad) == EINVAL
    for plan in (3, 8):
        assert _gemm(out_dtype=E4M3, c_scales=FAKE, ld_cs=1, plan=plan) == EUNSUPPORTED and "0 to 2" in _said()


@pytest.mark.parametrize("m", [(1 << 31) - 1, (1 << 31) - 16, (1 << 31) - 255])
@pytest.mark.parametrize("plan", [-1, 0, 4, 7])
def test_gemm_refuses_rows_that_tiles_cannot_count(m, plan):
    """Row counts whose rounding up to a whole tile (256 rows at most) passes
    31 bits are refused: tiles are counted in 32-bit integers."""
    assert _gemm(m=m, n=4, k=16, lda=16, ldw=16, ldc=4, ld_as=1, ld_ws=1, plan=plan) == EUNSUPPORTED
    assert "rows" in _said()

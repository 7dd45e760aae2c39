"""Calls of the residual branch's operators with arguments that make no sense end with an exception or a status, never with the process
(no GPU needed)."""
import ctypes

import pytest
import torch

from test_token_refusals import ALIGN, ARG, CAPACITY, DTYPE, NULL, SHAPE, changed


@pytest.fixture(scope="module")
def lib(built_library):
    from actnn_b200 import _lib
    return _lib.load()


def test_fp8_codes(lib):
    # x codes scales, rows cols ld_x ld_codes dtype, stream
    args, call = [256, 256, 256, 4, 40, 40, 48, 1, None], lib.actnn_fp8_row_codes
    assert call(*changed(args, _3=-1)) == SHAPE and call(*changed(args, _4=-1)) == SHAPE and call(*changed(args, _5=39)) == SHAPE
    assert call(*changed(args, _6=40)) == SHAPE and call(*changed(args, _6=64)) == SHAPE and call(*changed(args, _4=1 << 40)) == SHAPE
    assert call(*changed(args, _7=3)) == DTYPE and call(*changed(args, _3=0)) == 0 and call(*changed(args, _4=0, _6=0)) == 0
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in range(3))
    assert call(*changed(args, _0=257)) == ALIGN and call(*changed(args, _1=264)) == ALIGN and call(*changed(args, _2=264)) == ALIGN
    # x codes scales codes_t scales_t parts, rows cols ld_x ld_codes ld_codes_t square dtype, stream
    args, call = [256] * 6 + [20, 40, 40, 48, 32, 0, 1, None], lib.actnn_fp8_tile_codes
    assert call(*changed(args, _6=-1)) == SHAPE and call(*changed(args, _8=39)) == SHAPE and call(*changed(args, _9=64)) == SHAPE
    assert call(*changed(args, _10=16)) == SHAPE and call(*changed(args, _11=2)) == ARG and call(*changed(args, _12=3)) == DTYPE
    assert call(*changed(args, _6=0, _10=0)) == 0 and call(*changed(args, _1=None, _3=None, _5=None)) == NULL
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in (0, 2, 4))
    assert all(call(*changed(args, **{"_%d" % i: 264})) == ALIGN for i in (1, 2, 3, 4)) and call(*changed(args, _5=258)) == ALIGN
    # parts out, runs cols dtype, stream
    args, call = [256, 256, 3, 40, 1, None], lib.actnn_fp8_join_sums
    assert call(*changed(args, _2=-1)) == SHAPE and call(*changed(args, _4=9)) == DTYPE and call(*changed(args, _3=0)) == 0
    assert call(*changed(args, _0=None)) == NULL and call(*changed(args, _1=None)) == NULL and call(*changed(args, _1=257)) == ALIGN
    # codes scales out, rows cols ld_codes dtype, stream
    args, call = [256, 256, 256, 4, 40, 48, 1, None], lib.actnn_fp8_decode
    assert call(*changed(args, _3=-1)) == SHAPE and call(*changed(args, _5=39)) == SHAPE and call(*changed(args, _6=-1)) == DTYPE
    assert call(*changed(args, _4=0)) == 0 and all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in range(3))
    assert call(*changed(args, _2=257)) == ALIGN


def test_fp8_product(lib):
    # tokens token_scales weights weight_scales bias out, T N K ld_tokens ld_weights dtype, stream
    args, call = [256] * 6 + [4, 8, 40, 48, 48, 1, None], lib.actnn_fp8_matmul
    assert call(*changed(args, _6=-1)) == SHAPE and call(*changed(args, _8=0)) == SHAPE and call(*changed(args, _8=1 << 31)) == SHAPE
    assert call(*changed(args, _9=32)) == SHAPE and call(*changed(args, _10=39)) == SHAPE and call(*changed(args, _11=9)) == DTYPE
    assert call(*changed(args, _6=0)) == 0 and call(*changed(args, _7=0)) == 0
    assert call(*changed(args, _6=0x7fffff00, _7=0x7fffff00)) == SHAPE
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in (0, 1, 2, 3, 5))
    assert call(*changed(args, _0=264)) == ALIGN and call(*changed(args, _2=257)) == ALIGN and call(*changed(args, _9=50)) == ALIGN
    assert call(*changed(args, _1=264)) == ALIGN and call(*changed(args, _3=264)) == ALIGN
    assert call(*changed(args, _4=257)) == ALIGN and call(*changed(args, _5=257)) == ALIGN
    size = ctypes.c_int64(-1)
    need = lambda t, k: lib.actnn_fp8_linear_workspace(t, k, ctypes.addressof(size))          # noqa: E731
    assert need(1, 2048) == 0 and size.value == 0 and need(8, 4096) == 0 and size.value == 0
    assert need(100, 40) == 0 and size.value == 4864 + 512                # codes up to 256 bytes, scales of 128 rows and four blocks
    assert need(8, 8192) == 0 and size.value > 0                          # the codes of all do not fit shared memory
    assert need(1, 0) == SHAPE and need(-1, 8) == SHAPE and lib.actnn_fp8_linear_workspace(1, 8, None) == NULL
    # x weights weight_scales bias out, T N K ld_x ld_weights dtype, workspace bytes, stream
    args, call = [256] * 5 + [100, 8, 40, 40, 48, 1, 256, 5376, None], lib.actnn_fp8_linear
    assert call(*changed(args, _7=0)) == SHAPE and call(*changed(args, _8=39)) == SHAPE and call(*changed(args, _9=39)) == SHAPE
    assert call(*changed(args, _10=4)) == DTYPE and call(*changed(args, _5=0)) == 0
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in (0, 1, 2, 4, 11))
    assert call(*changed(args, _12=5375)) == CAPACITY and call(*changed(args, _11=264)) == ALIGN
    assert call(*changed(args, _0=257)) == ALIGN and call(*changed(args, _1=264)) == ALIGN and call(*changed(args, _9=56)) == ALIGN
    assert call(*changed(args, _2=264)) == ALIGN


def test_seeded_dropout(lib):
    # x y, numel p dtype seed offset state, stream
    args, call = [256, 256, 100, 0.5, 1, 1, 4, None, None], lib.actnn_seeded_dropout
    assert call(*changed(args, _2=-1)) == SHAPE and call(*changed(args, _4=3)) == DTYPE and call(*changed(args, _2=0)) == 0
    assert all(call(*changed(args, _3=p)) == ARG for p in (1.0, -0.1, 1.5, float("nan")))
    assert call(*changed(args, _0=None)) == NULL and call(*changed(args, _1=None)) == NULL
    assert call(*changed(args, _0=264)) == ALIGN and call(*changed(args, _1=264)) == ALIGN and call(*changed(args, _7=264)) == ALIGN
    assert lib.actnn_philox_state(None, 256, 0, 256, None) == NULL and lib.actnn_philox_state(256, 256, 0, 257, None) == ALIGN


def test_residual_norm(lib):
    size = ctypes.c_int64(0)
    call = lib.actnn_residual_norm_workspace
    assert call(-1, 8, 1, 0, ctypes.addressof(size)) == SHAPE and call(4, 32769, 1, 0, ctypes.addressof(size)) == SHAPE
    assert call(4, 8, 3, 0, ctypes.addressof(size)) == SHAPE and call(4, 8, 0, 0, ctypes.addressof(size)) == SHAPE and call(4, 8, 1, 0, None) == NULL
    assert call(1 << 31, 8, 1, 0, ctypes.addressof(size)) == SHAPE and call(8, 40, 4, 1, ctypes.addressof(size)) == 0 and size.value > 0
    # x f weight bias post_weight post_bias gate r h codes_x codes_f scale_x scale_f stats, rows C gate_rows scale eps layer post p dtype
    # param_dtype gate_dtype seed offset state, stream
    args, call = [256] * 14 + [8, 40, 4, 1.0, 1e-5, 1, 1, 0.1, 1, 1, 1, 1, 4, None, None], lib.actnn_residual_norm_forward
    assert call(*changed(args, _14=-1)) == SHAPE and call(*changed(args, _15=0)) == SHAPE and call(*changed(args, _16=3)) == SHAPE
    assert call(*changed(args, _18=-1.0)) == ARG and call(*changed(args, _18=float("nan"))) == ARG and call(*changed(args, _19=2)) == ARG
    assert call(*changed(args, _20=2)) == ARG and call(*changed(args, _21=1.0)) == ARG and call(*changed(args, _19=0)) == ARG     # rms with biases
    assert call(*changed(args, _20=0)) == ARG                              # parameters of a norm that is left out
    assert all(call(*changed(args, **{"_%d" % i: 3})) == DTYPE for i in (22, 23, 24)) and call(*changed(args, _14=0)) == 0
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in (0, 1, 7, 8, 9, 10, 11, 12, 13))
    assert all(call(*changed(args, **{"_%d" % i: 257})) == ALIGN for i in (0, 1, 2, 3, 4, 5, 6, 7, 8, 13)) and call(*changed(args, _27=264)) == ALIGN
    # grad_r grad_h x f codes_x codes_f scale_x scale_f stats weight post_weight post_bias gate grad_x grad_f grad_weight grad_bias
    # grad_post_weight grad_post_bias grad_gate, rows C gate_rows scale layer post p dtype param_dtype gate_dtype seed offset state,
    # workspace bytes stream
    args, call = [256] * 20 + [8, 40, 4, 1.0, 1, 1, 0.1, 1, 1, 1, 1, 4, None, 256, size.value, None], lib.actnn_residual_norm_backward
    assert call(*changed(args, _20=-1)) == SHAPE and call(*changed(args, _24=0)) == ARG and call(*changed(args, _25=0)) == ARG
    assert call(*changed(args, _26=-0.5)) == ARG and call(*changed(args, _28=7)) == DTYPE and call(*changed(args, _8=None)) == NULL
    assert call(*changed(args, _4=None)) == NULL and call(*changed(args, _6=None)) == NULL and call(*changed(args, _33=None)) == NULL
    assert call(*changed(args, _2=None, _4=None, _5=None)) == NULL and call(*changed(args, _34=size.value - 1)) == CAPACITY
    assert all(call(*changed(args, **{"_%d" % i: 257})) == ALIGN for i in (0, 1, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19, 33))


def test_python_entry_points_refuse_what_is_not_on_a_gpu():
    import actnn_b200 as actnn
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import fp8, residual_norm, seeded_dropout
    x, codes, scales = torch.zeros(4, 16), torch.zeros(8, 16, dtype=torch.float8_e4m3fn), torch.zeros(1, 1, 512, dtype=torch.uint8)
    for call in (lambda: fp8.quantize(x), lambda: fp8.quantize_weight(x), lambda: fp8.tile_codes(x), lambda: fp8.dequantize(codes, scales),
                 lambda: fp8.linear(x, codes, scales), lambda: fp8.matmul(codes, scales, codes, scales), lambda: ops.fp8_linear.apply(x, torch.zeros(8, 16)),
                 lambda: actnn.QFp8Linear(16, 8)(x), lambda: actnn.QFp8Linear(16, 8).freeze(), lambda: seeded_dropout.apply_mask(x, 0.5, (1, 2)),
                 lambda: ops.seeded_dropout.apply(x, 0.5), lambda: ops.seeded_dropout.apply(x, 0.5, (1, 4)), lambda: actnn.QSeededDropout()(x),
                 lambda: residual_norm.inference(x, x), lambda: residual_norm.run(x, x), lambda: ops.residual_norm.apply(x, x),
                 lambda: ops.residual_norm.apply(x.requires_grad_(), x), lambda: actnn.QResidualNorm(16)(x, x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_python_entry_points_refuse_numbers_that_make_no_sense():
    import actnn_b200 as actnn
    from actnn_b200 import ops
    x = torch.zeros(4, 16)
    for p in (1.0, -0.1, 2, float("nan"), "half"):
        for call in (lambda: ops.seeded_dropout.apply(x, p), lambda: ops.residual_norm.apply(x, x, p=p), lambda: actnn.QSeededDropout(p),
                     lambda: actnn.QResidualNorm(16, p=p)):
            with pytest.raises(RuntimeError, match="probability"):
                call()
    for key in (1, (1, 2, 3), (1.0, 2), "ab", (None, 4)):
        with pytest.raises(RuntimeError, match="key"):
            ops.seeded_dropout.apply(x, 0.5, key)
    with pytest.raises(RuntimeError, match="kind must be one of"):
        ops.residual_norm.apply(x, x, kind="group")
    with pytest.raises(RuntimeError, match="kind must be one of"):
        actnn.QResidualNorm(16, kind="group")

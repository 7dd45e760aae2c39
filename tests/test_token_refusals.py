"""Calls of the token operators with arguments that make no sense end with an exception or a status, never with the process
(no GPU needed)."""
import ctypes

import pytest
import torch

NULL, DTYPE, SHAPE, ALIGN, ARG, CAPACITY = 1, 2, 3, 5, 6, 8


@pytest.fixture(scope="module")
def lib(built_library):
    from actnn_b200 import _lib
    return _lib.load()


def changed(args, **at):
    args = list(args)
    for i, v in at.items():
        args[int(i[1:])] = v
    return args


def test_row_codes(lib):
    # x codes scale, rows cols ld_x ld_codes dtype, stream
    args, call = [256, 256, 256, 4, 40, 40, 48, 1, None], lib.actnn_row_codes
    assert call(*changed(args, _3=-1)) == SHAPE and call(*changed(args, _4=-1)) == SHAPE and call(*changed(args, _5=39)) == SHAPE
    assert call(*changed(args, _6=40)) == SHAPE and call(*changed(args, _6=64)) == SHAPE and call(*changed(args, _4=1 << 40)) == SHAPE
    assert call(*changed(args, _7=3)) == DTYPE and call(*changed(args, _3=0)) == 0
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in range(3))
    assert call(*changed(args, _0=257)) == ALIGN and call(*changed(args, _1=264)) == ALIGN and call(*changed(args, _2=258)) == ALIGN
    args, call = [256, 256, 256, 4, 40, 48, 1, None], lib.actnn_row_decode
    assert call(*changed(args, _3=-1)) == SHAPE and call(*changed(args, _5=39)) == SHAPE and call(*changed(args, _6=-1)) == DTYPE
    assert call(*changed(args, _4=0)) == 0 and all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in range(3))
    assert call(*changed(args, _2=257)) == ALIGN


def test_column_sums(lib):
    size = ctypes.c_int64(0)
    assert lib.actnn_column_sums_workspace(100, 40, ctypes.addressof(size)) == 0 and size.value > 0
    assert lib.actnn_column_sums_workspace(100, 40, None) == NULL and lib.actnn_column_sums_workspace(-1, 40, ctypes.addressof(size)) == SHAPE
    # x out, rows cols dtype, workspace bytes, stream
    args, call = [256, 256, 100, 40, 1, 256, 1 << 20, None], lib.actnn_column_sums
    assert call(*changed(args, _2=-1)) == SHAPE and call(*changed(args, _4=3)) == DTYPE and call(*changed(args, _3=0)) == 0
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in (0, 1, 5))
    assert call(*changed(args, _0=257)) == ALIGN and call(*changed(args, _5=258)) == ALIGN and call(*changed(args, _6=16)) == CAPACITY


def test_int8_matmul(lib):
    # tokens token_scale weights channel_scale bias out, T N K ld_tokens ld_weights dtype, stream
    args, call = [256] * 6 + [4, 8, 40, 48, 48, 1, None], lib.actnn_int8_matmul
    assert call(*changed(args, _6=-1)) == SHAPE and call(*changed(args, _8=0)) == SHAPE and call(*changed(args, _8=131073)) == SHAPE
    assert call(*changed(args, _9=32)) == SHAPE and call(*changed(args, _10=39)) == SHAPE and call(*changed(args, _11=9)) == DTYPE
    assert call(*changed(args, _6=0)) == 0 and call(*changed(args, _7=0)) == 0
    assert call(*changed(args, _6=0x7fffff00, _7=0x7fffff00)) == SHAPE
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in (0, 1, 2, 3, 5))
    assert call(*changed(args, _0=264)) == ALIGN and call(*changed(args, _2=257)) == ALIGN and call(*changed(args, _9=50)) == ALIGN
    assert call(*changed(args, _4=257)) == ALIGN and call(*changed(args, _5=257)) == ALIGN


def test_int8_linear(lib):
    size = ctypes.c_int64(-1)
    need = lambda t, k: lib.actnn_int8_linear_workspace(t, k, ctypes.addressof(size))          # noqa: E731
    assert need(1, 2048) == 0 and size.value == 0
    assert need(100, 40) == 0 and size.value == 100 * 48 + 400
    assert need(2, 131072) == 0 and size.value > 0                        # the codes of both do not fit shared memory
    assert need(1, 0) == SHAPE and need(-1, 8) == SHAPE and lib.actnn_int8_linear_workspace(1, 8, None) == NULL
    # x weights channel_scale bias out, T N K ld_x ld_weights dtype, workspace bytes, stream
    args, call = [256] * 5 + [100, 8, 40, 40, 48, 1, 256, 5200, None], lib.actnn_int8_linear
    assert call(*changed(args, _7=131073)) == SHAPE and call(*changed(args, _8=39)) == SHAPE and call(*changed(args, _9=39)) == SHAPE
    assert call(*changed(args, _10=4)) == DTYPE and call(*changed(args, _5=0)) == 0
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in (0, 1, 2, 4, 11))
    assert call(*changed(args, _12=5199)) == CAPACITY and call(*changed(args, _11=264)) == ALIGN
    assert call(*changed(args, _0=257)) == ALIGN and call(*changed(args, _1=264)) == ALIGN and call(*changed(args, _9=56)) == ALIGN


def test_activations(lib):
    # x y codes scale, rows cols gated kind dtype, stream
    args, call = [256] * 4 + [4, 40, 0, 2, 1, None], lib.actnn_act_forward
    assert call(*changed(args, _4=-1)) == SHAPE and call(*changed(args, _4=1 << 41, _5=1 << 41)) == SHAPE
    assert call(*changed(args, _6=2)) == ARG and call(*changed(args, _7=5)) == ARG and call(*changed(args, _7=-1)) == ARG
    assert call(*changed(args, _8=3)) == DTYPE and call(*changed(args, _4=0)) == 0
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in range(4))          # codes without scales, too
    assert call(*changed(args, _0=264)) == ALIGN and call(*changed(args, _2=260)) == ALIGN and call(*changed(args, _0=257, _6=1)) == ALIGN
    # grad_y x codes scale grad_x, rows cols gated kind dtype, stream
    args, call = [256] * 5 + [4, 40, 1, 2, 1, None], lib.actnn_act_backward
    assert call(*changed(args, _1=None, _2=None, _3=None)) == NULL and call(*changed(args, _0=None)) == NULL
    assert call(*changed(args, _3=None)) == NULL and call(*changed(args, _4=None)) == NULL and call(*changed(args, _4=257)) == ALIGN
    assert call(*changed(args, _9=7)) == DTYPE


def test_group_norm(lib):
    size = ctypes.c_int64(0)
    call = lib.actnn_group_norm_workspace
    assert call(2, 10, 16, 5, ctypes.addressof(size)) == SHAPE and call(2, 10, 16, 4, None) == NULL and call(2, 10, 0, 1, ctypes.addressof(size)) == SHAPE
    assert call(2, 10, 16, 4, ctypes.addressof(size)) == 0 and size.value > 0
    # x gamma beta y codes stats, N S C G eps kind dtype, workspace bytes, stream
    args, call = [256] * 6 + [2, 10, 16, 4, 1e-5, 2, 1, 256, size.value, None], lib.actnn_group_norm_forward
    assert call(*changed(args, _9=5)) == SHAPE and call(*changed(args, _6=-1)) == SHAPE and call(*changed(args, _9=0)) == SHAPE
    assert call(*changed(args, _10=-1.0)) == ARG and call(*changed(args, _10=float("nan"))) == ARG and call(*changed(args, _11=9)) == ARG
    assert call(*changed(args, _12=3)) == DTYPE and call(*changed(args, _6=0)) == 0 and call(*changed(args, _7=0)) == 0
    assert all(call(*changed(args, **{"_%d" % i: None})) == NULL for i in (0, 3, 5, 13))
    assert call(*changed(args, _0=257)) == ALIGN and call(*changed(args, _13=264)) == ALIGN and call(*changed(args, _5=260)) == ALIGN
    assert call(*changed(args, _14=size.value - 1)) == CAPACITY
    # grad_y x codes stats gamma beta grad_x grad_gamma grad_beta, N S C G kind dtype, workspace bytes, stream
    args, call = [256] * 9 + [2, 10, 16, 4, 2, 1, 256, size.value, None], lib.actnn_group_norm_backward
    assert call(*changed(args, _1=None, _2=None)) == NULL and call(*changed(args, _3=None)) == NULL and call(*changed(args, _6=None)) == NULL
    assert call(*changed(args, _13=-2)) == ARG and call(*changed(args, _14=5)) == DTYPE and call(*changed(args, _16=0)) == CAPACITY
    assert call(*changed(args, _6=257)) == ALIGN


def test_python_entry_points_refuse_what_is_not_on_a_gpu():
    import actnn_b200 as actnn
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import checkpoint, group_norm, int8
    x, codes = torch.zeros(4, 16), torch.zeros(8, 16, dtype=torch.int8)
    for call in (lambda: int8.quantize_rows(x), lambda: int8.linear(x, codes, torch.zeros(8)), lambda: int8.dequantize_rows(codes, torch.zeros(8)),
                 lambda: int8.matmul(codes, torch.zeros(8), codes, torch.zeros(8)), lambda: checkpoint.activation_forward(x, "silu"),
                 lambda: checkpoint.activation_backward(x, "silu", x=x), lambda: group_norm.inference(x, 4), lambda: group_norm.forward(x, 4),
                 lambda: ops.activation.apply(x, "silu"), lambda: ops.glu.apply(x, "silu"), lambda: ops.group_norm.apply(x, 4),
                 lambda: ops.int8_linear.apply(x, torch.zeros(8, 16)), lambda: actnn.QSiLU()(x), lambda: actnn.QInt8Linear(16, 8)(x),
                 lambda: actnn.QGroupNorm(4, 16)(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="activation must be one of"):
        ops.activation.apply(x, "swish")
    with pytest.raises(RuntimeError, match="activation must be one of"):
        actnn.QGLU("swish")

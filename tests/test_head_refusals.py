"""The training head's argument checks: everything here is refused on the host, before any HIP call."""
import ctypes
import math

import pytest
import torch

from recsdk_amd import capi, torch_ops

F32, BF16, F16, I64 = capi.DT_F32, capi.DT_BF16, capi.DT_F16, capi.DT_I64
SOME = 4096   # stands for a device pointer; the calls are refused before it is used


def text():
    return capi.lib().recsdk_last_error().decode()


@pytest.mark.parametrize("args,code,word", [
    ((SOME, 8, I64, 0.5, 0, 0, None, SOME, None), capi.EINVAL, "dtype"),
    ((SOME, 8, F32, -0.1, 0, 0, None, SOME, None), capi.EINVAL, "p must"),
    ((SOME, 8, F32, 1.1, 0, 0, None, SOME, None), capi.EINVAL, "p must"),
    ((SOME, 8, F32, float("nan"), 0, 0, None, SOME, None), capi.EINVAL, "p must"),
    ((SOME, -1, F32, 0.5, 0, 0, None, SOME, None), capi.EINVAL, "negative"),
    ((None, 8, F32, 0.5, 0, 0, None, SOME, None), capi.ENULL, "NULL"),
    ((SOME, 8, F32, 0.5, 0, 0, None, None, None), capi.ENULL, "NULL"),
    ((SOME + 2, 8, F32, 0.5, 0, 0, None, SOME, None), capi.EINVAL, "aligned"),
    ((SOME + 1, 8, BF16, 0.5, 0, 0, None, SOME, None), capi.EINVAL, "aligned"),
    ((SOME, 2 ** 62, F32, 0.5, 0, 0, None, SOME, None), capi.EINVAL, "too large"),
])
def test_dropout(args, code, word):
    assert capi.lib().recsdk_dropout(*args) == code and word in text()


@pytest.mark.parametrize("args,code,word", [
    ((SOME, 4, 8, 8, I64, None, None, F32, 1e-5, SOME, None, None, None), capi.EINVAL, "dtype"),
    ((SOME, 4, 8, 8, F32, None, None, BF16, 1e-5, SOME, None, None, None), capi.EINVAL, "weight"),
    ((SOME, 4, 8, 8, BF16, None, None, F16, 1e-5, SOME, None, None, None), capi.EINVAL, "weight"),
    ((SOME, 4, 0, 8, F32, None, None, F32, 1e-5, SOME, None, None, None), capi.EINVAL, "dim"),
    ((SOME, -4, 8, 8, F32, None, None, F32, 1e-5, SOME, None, None, None), capi.EINVAL, "rows"),
    ((SOME, 2 ** 31, 8, 8, F32, None, None, F32, 1e-5, SOME, None, None, None), capi.EINVAL, "rows"),
    ((SOME, 4, 8, 7, F32, None, None, F32, 1e-5, SOME, None, None, None), capi.EINVAL, "overlap"),
    ((SOME, 4, 8, 8, F32, None, None, F32, -1.0, SOME, None, None, None), capi.EINVAL, "eps"),
    ((SOME, 4, 8, 8, F32, None, None, F32, float("nan"), SOME, None, None, None), capi.EINVAL, "eps"),
    ((SOME, 4, 8, 8, F32, None, None, F32, 1e-5, SOME, SOME, None, None), capi.EINVAL, "together"),
    ((None, 4, 8, 8, F32, None, None, F32, 1e-5, SOME, None, None, None), capi.ENULL, "NULL"),
    ((SOME, 4, 8, 8, F32, None, None, F32, 1e-5, None, None, None, None), capi.ENULL, "NULL"),
])
def test_layer_norm_forward(args, code, word):
    assert capi.lib().recsdk_layer_norm_forward(*args) == code and word in text()


@pytest.mark.parametrize("change,code,word", [
    (dict(grad=None), capi.ENULL, "NULL"), (dict(mean=None), capi.ENULL, "NULL"), (dict(dtype=I64), capi.EINVAL, "dtype"),
    (dict(stride=7), capi.EINVAL, "overlap"), (dict(space=None), capi.ECAPACITY, "workspace"),
    (dict(size=4 * 2 * 8 * 4 - 1), capi.ECAPACITY, "workspace"), (dict(space=SOME + 8), capi.EINVAL, "aligned"),
])
def test_layer_norm_backward(change, code, word):
    a = dict(grad=SOME, x=SOME, rows=4, dim=8, stride=8, dtype=F32, weight=None, wtype=F32, mean=SOME, rstd=SOME, dx=SOME, dw=SOME,
             db=SOME, space=SOME, size=1 << 20, stream=None)
    assert capi.lib().recsdk_layer_norm_backward(*{**a, **change}.values()) == code and word in text()


def test_layer_norm_workspace():
    n = ctypes.c_int64()
    assert capi.lib().recsdk_layer_norm_workspace(4, 8, None) == capi.ENULL
    assert capi.lib().recsdk_layer_norm_workspace(4, 0, n) == capi.EINVAL
    assert capi.lib().recsdk_layer_norm_workspace(4, 8, n) == capi.OK and n.value == 4 * 2 * 8 * 4
    assert capi.lib().recsdk_layer_norm_workspace(0, 8, n) == capi.OK and n.value == 0


SIZES = dict(rows=4, items=9, dim=8, dtype=F32, x_stride=8, table_stride=8)
BAD_SIZES = [(dict(dtype=F16), "fp32 or bf16"), (dict(dim=0), "dim"), (dict(dim=257, x_stride=300, table_stride=300), "dim"),
             (dict(rows=-1), "rows"), (dict(rows=2 ** 30), "rows"), (dict(items=0), "items"), (dict(items=2 ** 30), "items"),
             (dict(x_stride=7), "overlap"), (dict(table_stride=7), "overlap")]


@pytest.mark.parametrize("change,word", BAD_SIZES)
def test_softmax_loss_sizes(change, word):
    L, f, b = capi.lib(), ctypes.c_int64(), ctypes.c_int64()
    s = {**SIZES, **change}
    assert L.recsdk_softmax_loss_workspace(*s.values(), f, b) == capi.EINVAL and word in text()
    args = (SOME, s["rows"], s["x_stride"], SOME, s["items"], s["table_stride"], s["dim"], s["dtype"], SOME, None, 1.0)
    assert L.recsdk_softmax_loss_forward(*args, SOME, SOME, SOME, 1 << 30, None) == capi.EINVAL and word in text()
    assert L.recsdk_softmax_loss_backward(SOME, *args, SOME, SOME, SOME, SOME, 1 << 30, None) == capi.EINVAL and word in text()


@pytest.mark.parametrize("change,code,word", [
    (dict(x=None), capi.ENULL, "NULL"), (dict(table=None), capi.ENULL, "NULL"), (dict(target=None), capi.ENULL, "NULL"),
    (dict(x=SOME + 4), capi.EINVAL, "aligned"), (dict(table=SOME + 8), capi.EINVAL, "aligned"),
    (dict(space=SOME + 8), capi.EINVAL, "aligned"), (dict(space=None), capi.ECAPACITY, "workspace"),
    (dict(size=16), capi.ECAPACITY, "workspace"),
])
def test_softmax_loss_pointers(change, code, word):
    L = capi.lib()
    a = {**dict(x=SOME, table=SOME, target=SOME, space=SOME, size=1 << 30), **change}
    args = (a["x"], 4, 8, a["table"], 9, 8, 8, F32, a["target"], None, 1.0)
    assert L.recsdk_softmax_loss_forward(*args, SOME, SOME, a["space"], a["size"], None) == code and word in text()
    assert L.recsdk_softmax_loss_backward(SOME, *args, SOME, SOME, SOME, a["space"], a["size"], None) == code and word in text()
    assert L.recsdk_softmax_loss_backward(SOME, *args, SOME, None, None, None, 0, None) == capi.OK   # nothing wanted


def test_softmax_loss_workspace_grows_with_what_is_copied():
    L, f, b = capi.lib(), ctypes.c_int64(), ctypes.c_int64()
    assert L.recsdk_softmax_loss_workspace(100, 1000, 64, BF16, 64, 64, f, b) == capi.OK
    plain = f.value, b.value
    assert L.recsdk_softmax_loss_workspace(100, 1000, 64, BF16, 64, 65, f, b) == capi.OK   # off the 16-byte border: read as they are
    assert (f.value, b.value) == plain
    assert L.recsdk_softmax_loss_workspace(100, 1000, 8, BF16, 8, 8, f, b) == capi.OK
    plain = f.value, b.value
    assert L.recsdk_softmax_loss_workspace(100, 1000, 7, BF16, 7, 7, f, b) == capi.OK   # shorter than a 16-byte piece: copied
    assert f.value >= plain[0] + 1000 * 8 * 2 and b.value >= plain[1] + 1000 * 8 * 2
    assert L.recsdk_softmax_loss_workspace(0, 1000, 64, BF16, 64, 64, f, b) == capi.OK and f.value == b.value == 0


@pytest.mark.parametrize("dtype,bias,scale", [(F32, None, math.inf), (BF16, None, -math.inf), (F32, SOME, math.nan), (BF16, SOME, 1e-13),
                                              (BF16, SOME, -1e-30)])
def test_softmax_loss_scales(dtype, bias, scale):
    L = capi.lib()
    args = (SOME, 4, 8, SOME, 9, 8, 8, dtype, SOME, bias, scale)
    assert L.recsdk_softmax_loss_forward(*args, SOME, SOME, SOME, 1 << 30, None) == capi.EINVAL and "scale" in text()
    assert L.recsdk_softmax_loss_backward(SOME, *args, SOME, SOME, SOME, SOME, 1 << 30, None) == capi.EINVAL and "scale" in text()


def test_softmax_loss_rows_far_apart_are_copied():
    L, f, b = capi.lib(), ctypes.c_int64(), ctypes.c_int64()
    assert L.recsdk_softmax_loss_workspace(100, 1000, 64, F32, 64, 2 ** 22, f, b) == capi.OK
    near = f.value, b.value
    assert L.recsdk_softmax_loss_workspace(100, 1000, 64, F32, 64, 2 ** 22 + 4, f, b) == capi.OK
    assert f.value >= near[0] + 1000 * 64 * 4 and b.value >= near[1] + 1000 * 64 * 4


def test_layer_norm_rows_too_long():
    n = ctypes.c_int64()
    assert capi.lib().recsdk_layer_norm_workspace(4, 2 ** 30, n) == capi.EINVAL
    args = (SOME, 1, 2 ** 30, 2 ** 30, F32, None, None, F32, 1e-5, SOME, None, None, None)
    assert capi.lib().recsdk_layer_norm_forward(*args) == capi.EINVAL and "dim" in text()


def test_host_tensors_are_refused():
    torch_ops.load()
    ops = torch.ops.recsdk
    x, table, target = torch.zeros(4, 8), torch.zeros(9, 8), torch.zeros(4, dtype=torch.long)
    for call in (lambda: ops.dropout(x, 0.5, 1), lambda: ops.layer_norm(x), lambda: ops.softmax_loss(x, table, target)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_operators_are_registered():
    torch_ops.load()
    for name, arguments in {"dropout": 5, "layer_norm": 4, "layer_norm_forward": 4, "layer_norm_backward": 6, "softmax_loss": 5,
                            "softmax_loss_forward": 5, "softmax_loss_backward": 8}.items():
        assert len(getattr(torch.ops.recsdk, name).default._schema.arguments) == arguments

"""GPU: the training head (dropout, layer norm, softmax loss over a table) through the torch operators and the C ABI,
against plain forms in 64 bits."""
import ctypes
import math

import pytest
import torch

from recsdk_amd import capi, host, torch_ops
from tests import head_cases as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    torch_ops.load()
    return torch.ops.recsdk


def randn(*shape, seed=0, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


# ---- dropout ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 4095, 4096, 4104, 100003])
def test_dropout_matches_the_generator(ops, kind, n):
    x = randn(n, seed=n, dtype=TYPES[kind])
    for p, seed, offset in ((0.1, 3, 0), (0.5, -1, 2 ** 40 + 3), (0.9, 2 ** 62 + 17, -5)):
        want, keep = plain.dropout(x, p, seed, offset)
        assert torch.equal(ops.dropout(x, p, seed, offset).cpu(), want)
    assert n < 4000 or abs(keep.double().mean().item() - 0.1) < 5 * math.sqrt(0.09 / n)


def test_dropout_ends_of_the_range_and_dropped_infinities(ops):
    x = randn(1000, seed=1)
    assert torch.equal(ops.dropout(x, 0.0, 5), x)
    assert torch.equal(ops.dropout(x, 1.0, 5), torch.zeros_like(x))
    bad = torch.full_like(x, math.nan)
    bad[::2] = math.inf
    y = ops.dropout(bad, 0.5, 5).cpu()
    _, keep = plain.dropout(x, 0.5, 5, 0)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    assert ops.dropout(x[:0], 0.5, 1).shape == (0,)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_dropout_gradient_uses_the_same_mask(ops, kind):
    x = randn(37, 51, seed=2, dtype=TYPES[kind]).requires_grad_()
    grad = randn(37, 51, seed=3, dtype=TYPES[kind])
    y = ops.dropout(x, 0.3, 11, 7)
    (dx,) = torch.autograd.grad(y, (x,), grad)
    assert torch.equal(dx.cpu(), plain.dropout(grad, 0.3, 11, 7)[0])
    # a gradient with strides of its own, as a broadcast sum has
    y = ops.dropout(x, 0.3, 11, 7)
    (dx,) = torch.autograd.grad(y.sum(), (x,))
    assert torch.equal(dx.cpu(), plain.dropout(torch.ones_like(grad), 0.3, 11, 7)[0])


def test_dropout_of_views_and_odd_addresses(ops):
    base = randn(4001, seed=4, dtype=torch.bfloat16)
    for lo in (1, 3, 8):
        x = base[lo:lo + 1003]
        assert torch.equal(ops.dropout(x, 0.4, 9).cpu(), plain.dropout(x, 0.4, 9, 0)[0])
    x = randn(20, 30, seed=5).t()
    assert torch.equal(ops.dropout(x, 0.4, 9).cpu(), plain.dropout(x.contiguous(), 0.4, 9, 0)[0])


def test_dropout_in_place_through_the_c_abi():
    x = randn(5000, seed=6)
    want = plain.dropout(x, 0.25, 1, 2)[0]
    capi.check(capi.lib().recsdk_dropout(x.data_ptr(), x.numel(), capi.DT_F32, 0.25, 1, 2, None, x.data_ptr(),
                                         host._stream()))
    assert torch.equal(x.cpu(), want)


def test_dropout_step_word_moves_the_mask_of_a_replayed_graph(ops):
    x = randn(3000, seed=7)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    ops.dropout(x, 0.5, 3, 10, step)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.dropout(x, 0.5, 3, 10, step)
        step.add_(1)
    step.zero_()
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), plain.dropout(x, 0.5, 3, 10 + k)[0])
        assert torch.equal(ops.dropout(x, 0.5, 3, 10 + k).cpu(), y.cpu())


def test_dropout_step_advanced_before_the_backward_pass_is_an_error(ops):
    x = randn(100, seed=8).requires_grad_()
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    y = ops.dropout(x, 0.5, 3, 0, step)
    step.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- layer norm ------------------------------------------------------------------------------------------------------

def norm_case(rows, dim, kind, wkind, seed, offset=3.0):
    x = (randn(rows, dim, seed=seed) + offset * randn(1, dim, seed=seed + 1)).to(TYPES[kind])
    weight = (1 + 0.1 * randn(dim, seed=seed + 2)).to(TYPES[wkind])
    bias = randn(dim, seed=seed + 3, std=0.1, dtype=TYPES[wkind])
    return x, weight, bias, randn(rows, dim, seed=seed + 4, dtype=TYPES[kind])


def check_norm(ops, x, weight, bias, grad, eps=1e-5):
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, weight, bias)]
    y = ops.layer_norm(*leaves, eps)
    wanted = [t for t in leaves if t is not None]
    got = torch.autograd.grad(y, wanted, grad)
    want = plain.layer_norm(x.reshape(-1, x.shape[-1]), weight, bias, eps, grad.reshape(-1, x.shape[-1]))
    plain.close(y.reshape(want[0][0].shape), want[0], "y")
    plain.close(got[0].reshape(want[1][0].shape), want[1], "dx")
    k = 1
    for t, w, name in ((weight, want[2], "dweight"), (bias, want[3], "dbias")):
        if t is not None:
            assert got[k].dtype == t.dtype
            plain.close(got[k], w, name)
            k += 1
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, weight, bias, eps), y)


# widths: one, odd ones, each team size, each number of packs, past the registers; 16-byte packs and single elements
@pytest.mark.parametrize("kind,wkind", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,dim", [(5, 1), (33, 7), (70, 16), (9, 36), (100, 64), (65, 100), (40, 128), (7, 201), (30, 256),
                                      (11, 500), (6, 1001), (12, 1664), (3, 3328), (2, 5003), (2, 8192), (1, 16384)])
def test_layer_norm_forward_and_gradients(ops, kind, wkind, rows, dim):
    check_norm(ops, *norm_case(rows, dim, kind, wkind, rows + dim))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [16400, 33000, 40001])
def test_layer_norm_rows_past_the_registers(ops, kind, dim):
    check_norm(ops, *norm_case(20, dim, kind, "f32", dim))


@pytest.mark.parametrize("rows,dim,kind", [(20000, 16, "f32"), (9001, 128, "bf16"), (3001, 1001, "f16"), (5000, 2048, "f32")])
def test_layer_norm_many_rows(ops, rows, dim, kind):
    check_norm(ops, *norm_case(rows, dim, kind, "f32", 77))


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
def test_layer_norm_without_parameters(ops, weight, bias):
    x, w, b, grad = norm_case(50, 72, "f32", "f32", 5)
    check_norm(ops, x, w if weight else None, b if bias else None, grad)
    x, w, b, grad = norm_case(50, 72, "bf16", "bf16", 5)
    check_norm(ops, x, w if weight else None, b if bias else None, grad)


def test_layer_norm_shapes_strides_and_odd_addresses(ops):
    x, w, b, grad = norm_case(60, 64, "bf16", "f32", 9)
    check_norm(ops, x.reshape(3, 4, 5, 64), w, b, grad.reshape(3, 4, 5, 64))
    check_norm(ops, x[0], w, b, grad[0])
    wide, _, _, _ = norm_case(60, 200, "bf16", "f32", 10)
    check_norm(ops, wide[:, :64], w, b, grad)          # rows of a wider matrix
    check_norm(ops, wide[:, 3:67], w, b, grad)         # that start off the 16-byte border
    check_norm(ops, wide[::3, 8:72], w, b, grad[:20])
    check_norm(ops, wide[:1].expand(60, 200)[:, :64], w, b, grad)
    check_norm(ops, randn(64, 60, seed=3, dtype=torch.bfloat16).t(), w, b, grad)
    check_norm(ops, x, w, b, grad[:1].expand(60, 64))


def test_layer_norm_empty_and_constant_rows(ops):
    x, w, b, _ = norm_case(4, 96, "f32", "f32", 11)
    leaves = [t.detach().requires_grad_() for t in (x[:0], w, b)]
    y = ops.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 96) and (dw == 0).all() and (db == 0).all()
    flat = torch.full((3, 96), 2.5, device=DEV)
    assert torch.equal(ops.layer_norm(flat, w, b), b.expand(3, 96))


def test_layer_norm_a_bad_row_stays_in_its_row(ops):
    x, w, b, grad = norm_case(50, 48, "f32", "f32", 12)
    x[7, 3], x[20, 5] = math.nan, math.inf
    y = ops.layer_norm(x, w, b)
    good = torch.ones(50, dtype=torch.bool)
    good[[7, 20]] = False
    assert torch.isnan(y[7]).all() and torch.isnan(y[20]).all()
    plain.close(y[good.to(DEV)], plain.layer_norm(x[good.to(DEV)], w, b, 1e-5)[0])


def test_layer_norm_is_repeatable_bit_for_bit(ops):
    x, w, b, grad = norm_case(4097, 100, "bf16", "f32", 13)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, 1e-5)
    first = ops.layer_norm_backward(grad, x, w, mean, rstd, [True, True, True])
    for _ in range(3):
        for a, c in zip(first, ops.layer_norm_backward(grad, x, w, mean, rstd, [True, True, True])):
            assert torch.equal(a, c)
    dx, none, also = ops.layer_norm_backward(grad, x, w, mean, rstd, [True, False, False])
    assert torch.equal(dx, first[0]) and (none is None or none.numel() == 0 or not none.defined())


# ---- softmax loss ----------------------------------------------------------------------------------------------------

def loss_case(rows, items, dim, kind, seed, std=0.7):
    x = randn(rows, dim, seed=seed, dtype=TYPES[kind])
    table = randn(items, dim, seed=seed + 1, std=std, dtype=TYPES[kind])
    target = torch.randint(0, items, (rows,), generator=torch.Generator().manual_seed(seed + 2)).to(DEV)
    grad = (0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(seed + 3))).to(DEV)
    return x, table, target, grad


def check_loss(ops, x, table, target, bias, scale, grad):
    leaves = [t.detach().requires_grad_() for t in (x, table)]
    loss = ops.softmax_loss(*leaves, target, bias, scale)
    dx, dt = torch.autograd.grad(loss, leaves, grad)
    want = plain.softmax_loss(x, table, target, bias, scale, grad)
    assert loss.dtype == torch.float32 and dx.dtype == x.dtype and dt.dtype == table.dtype
    plain.close(loss, want[0], "loss")
    plain.close(dx, want[1], "dx")
    plain.close(dt, want[2], "dtable")
    with torch.no_grad():
        assert torch.equal(ops.softmax_loss(x, table, target, bias, scale), loss)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [1, 16, 33, 64, 96, 100, 128, 160, 161, 192, 224, 225, 256])
def test_softmax_loss_widths_of_few_rows(ops, kind, dim):
    x, table, target, grad = loss_case(20, 333, dim, kind, dim)
    check_loss(ops, x, table, target, None, 3 / math.sqrt(dim), grad)
    bias = torch.randn(333, generator=torch.Generator().manual_seed(dim)).to(DEV)
    check_loss(ops, x, table, target, bias, 3 / math.sqrt(dim), grad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [72, 96, 129, 160, 192, 224])
def test_softmax_loss_widths_with_a_bias(ops, kind, dim):
    x, table, target, grad = loss_case(200, 333, dim, kind, dim)
    bias = torch.randn(333, generator=torch.Generator().manual_seed(dim)).to(DEV)
    bias[::7] = -math.inf
    check_loss(ops, x, table, target, bias, 3 / math.sqrt(dim), grad)


@pytest.mark.parametrize("big,small", [(1e15, 1e-15), (1e-18, 1e18), (1e-30, 1.0), (1e4, 1e4)])
def test_softmax_loss_magnitudes_of_float32(ops, big, small):
    x, table, target, grad = loss_case(100, 400, 64, "f32", 91)
    scale = 0.4 / (big * small)
    check_loss(ops, x * big, table * small, target, None, scale, grad)
    # rows of very different sizes: the smallest take part with 2^-22 of themselves as long as they are 2^-18 of the largest
    rise = torch.logspace(-4, 0, 400, device=DEV)[:, None]
    check_loss(ops, x * big, table * small * rise, target, None, scale, grad)


def test_softmax_loss_gradients_of_very_different_rows(ops):
    """Gradients of loss from 1e-12 to 1e6, also negative ones and zeros: every item keeps the precision of its own rows."""
    for kind in ("f32", "bf16"):
        x, table, target, grad = loss_case(300, 350, 48, kind, 92)
        grad = grad * torch.logspace(-12, 6, 300, device=DEV)
        grad[::3] *= -1
        grad[7::11] = 0
        order = torch.randperm(300, generator=torch.Generator().manual_seed(1)).to(DEV)
        for g in (grad, grad.flip(0).contiguous(), grad[order].contiguous()):
            check_loss(ops, x, table, target, None, 0.5, g)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [1, 7, 8, 16, 32, 36, 64, 68, 100, 128, 132, 200, 201, 255, 256])
def test_softmax_loss_widths(ops, kind, dim):
    x, table, target, grad = loss_case(70, 333, dim, kind, dim)
    check_loss(ops, x, table, target, None, 3 / math.sqrt(dim), grad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 64, 65, 127, 129, 257, 600])
@pytest.mark.parametrize("items,dim", [(1, 64), (2, 20), (31, 64), (33, 128), (64, 256), (65, 32), (129, 40), (1030, 64)])
def test_softmax_loss_row_and_item_counts(ops, kind, rows, items, dim):
    x, table, target, grad = loss_case(rows, items, dim, kind, rows * 7 + items)
    check_loss(ops, x, table, target, None, 0.4, grad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,items,dim", [(1, 700, 64), (40, 300, 24), (150, 1000, 128), (300, 257, 200)])
def test_softmax_loss_bias_free_slots_and_padding(ops, kind, rows, items, dim):
    x, table, target, grad = loss_case(rows, items, dim, kind, 3 * rows)
    g = torch.Generator().manual_seed(4)
    bias = torch.randn(items, generator=g).to(DEV)
    check_loss(ops, x, table, target, bias, 0.5, grad)
    # taken out by -infinity, by the type's lowest value and by anything below -1e30; their rows hold garbage
    for k, low in enumerate((-math.inf, torch.finfo(torch.float32).min, -1e30, -2e30)):
        bias[k::9] = low
    out = torch.where(bias <= -1e30)[0]
    table[out[::2]] = math.nan
    table[out[1::2]] = math.inf
    target[::5] = -1
    target[1::7] = items
    target[2::11] = -2 ** 40
    x[::5] = math.nan
    x[1::7] = math.inf
    grad[::5] = math.nan   # of rows that take none
    check_loss(ops, x, table, target, bias, 0.5, grad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_softmax_loss_rows_left_without_items(ops, kind):
    x, table, target, grad = loss_case(90, 50, 48, kind, 5)
    target[4] = -1
    check_loss(ops, x, table, target, torch.full((50,), -math.inf, device=DEV), 1.0, grad)
    bias = torch.full((50,), -math.inf, device=DEV)
    bias[17] = 0.5
    target[::2] = 17
    check_loss(ops, x, table, target, bias, 1.0, grad)   # one item left: loss 0, or infinite


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_softmax_loss_large_negative_zero_and_sharp_scores(ops, kind):
    x, table, target, grad = loss_case(130, 500, 64, kind, 6)
    for scale in (-0.6, 0.0, 12.0, 1e-4):
        check_loss(ops, x, table, target, None, scale, grad)
    bias = torch.full((500,), -1e4, device=DEV)   # far from zero, but nothing is taken out
    check_loss(ops, x, table, target, bias, 0.5, grad)
    # scores that rise along the table, so that the running maximum moves all the way; and fall
    ramp = torch.linspace(-300, 300, 500, device=DEV)
    for b in (ramp, ramp.flip(0).contiguous()):
        check_loss(ops, x, table, target, b, 0.5, grad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [20, 64, 90, 128, 200, 224, 256])
@pytest.mark.parametrize("rows", [6, 70, 300])
def test_softmax_loss_scales_with_a_bias(ops, kind, dim, rows):
    x, table, target, grad = loss_case(rows, 301, dim, kind, 20 + dim)
    bias = 5 * torch.randn(301, generator=torch.Generator().manual_seed(dim)).to(DEV)
    free = torch.arange(301, device=DEV) % 5 == 2
    bias[free] = -math.inf
    table[free] = math.nan
    target = torch.where(free[target], target - 1, target)
    for scale in (0.0, -0.3, 1e-6, 2.0 ** -40):
        check_loss(ops, x, table, target, bias, scale, grad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_softmax_loss_strided_rows(ops, kind):
    x, table, target, grad = loss_case(45, 400, 64, kind, 7)
    wide = randn(400, 192, seed=8, dtype=TYPES[kind])   # [row | state | state]: rows with optimizer state behind them
    wide[:, :64] = table
    check_loss(ops, x, wide[:, :64], target, None, 0.3, grad)
    wide[:, 5:69] = table
    check_loss(ops, x, wide[:, 5:69], target, None, 0.3, grad)   # rows off the 16-byte border
    odd = randn(400, 193, seed=9, dtype=TYPES[kind])
    odd[:, :64] = table
    check_loss(ops, x, odd[:, :64], target, None, 0.3, grad)     # a stride of no whole pieces
    check_loss(ops, x.t().contiguous().t(), table.t().contiguous().t(), target, None, 0.3, grad)
    check_loss(ops, x[::2], table[1::3], (target % 133)[::2], None, 0.3, grad[::2])
    check_loss(ops, x[:1].expand(45, 64), table, target.int(), None, 0.3, grad[:1].expand(45))


def test_softmax_loss_many_splits_and_rows(ops):
    x, table, target, grad = loss_case(3, 40000, 96, "bf16", 9)
    check_loss(ops, x, table, target, None, 0.5, grad)
    x, table, target, grad = loss_case(5000, 70, 64, "f32", 10)
    check_loss(ops, x, table, target, None, 0.5, grad)
    x, table, target, grad = loss_case(2100, 3000, 64, "bf16", 11)
    check_loss(ops, x, table, target, None, 0.5, grad)


def test_softmax_loss_gradient_against_differences(ops):
    x, table, target, grad = loss_case(9, 40, 16, "f32", 12)
    leaves = [t.detach().requires_grad_() for t in (x, table)]
    dx, dt = torch.autograd.grad((ops.softmax_loss(*leaves, target, None, 1.0) * grad).sum(), leaves)
    g = torch.Generator().manual_seed(13)
    for _ in range(4):
        vx, vt = torch.randn(9, 16, generator=g).to(DEV), torch.randn(40, 16, generator=g).to(DEV)
        step = 1e-2

        def at(s):
            return (ops.softmax_loss(x + s * vx, table + s * vt, target, None, 1.0).double() * grad.double()).sum().item()

        # fourth order: off by about step^4 times a fifth derivative, and by the loss's rounding over step
        slope = (8 * (at(step) - at(-step)) - (at(2 * step) - at(-2 * step))) / (12 * step)
        direct = ((dx * vx).double().sum() + (dt * vt).double().sum()).item()
        assert abs(slope - direct) < 5e-3 * max(1.0, abs(direct))


def test_softmax_loss_one_gradient_at_a_time_and_repeatable(ops):
    x, table, target, grad = loss_case(200, 900, 64, "bf16", 14)
    loss, lse = ops.softmax_loss_forward(x, table, target, None, 0.4)
    both = ops.softmax_loss_backward(grad, x, table, target, lse, None, 0.4, [True, True])
    for _ in range(3):
        again = ops.softmax_loss_backward(grad, x, table, target, lse, None, 0.4, [True, True])
        assert all(torch.equal(a, b) for a, b in zip(both, again))
    assert torch.equal(ops.softmax_loss_backward(grad, x, table, target, lse, None, 0.4, [True, False])[0], both[0])
    assert torch.equal(ops.softmax_loss_backward(grad, x, table, target, lse, None, 0.4, [False, True])[1], both[1])
    xg = x.detach().requires_grad_()
    ops.softmax_loss(xg, table, target, None, 0.4).backward(grad)
    assert torch.equal(xg.grad, both[0])


def test_softmax_loss_of_no_rows(ops):
    x, table, target, grad = loss_case(3, 20, 64, "f32", 15)
    leaves = [t.detach().requires_grad_() for t in (x[:0], table)]
    loss = ops.softmax_loss(*leaves, target[:0])
    dx, dt = torch.autograd.grad(loss, leaves, grad[:0])
    assert loss.shape == (0,) and dx.shape == (0, 64) and dt.shape == table.shape and (dt == 0).all()


def test_softmax_loss_a_nan_row_is_seen(ops):
    x, table, target, grad = loss_case(70, 90, 32, "f32", 16)
    x[5, 3] = math.nan
    loss = ops.softmax_loss(x, table, target)
    assert torch.isnan(loss[5]) and torch.isfinite(loss[[0, 4, 6, 69]]).all()


def test_softmax_loss_table_past_32_bit_offsets(ops):
    # 17 M rows of 256 columns: 4.4e9 elements; all items but a few at both ends are taken out
    items, dim = 17_000_000, 256
    table = torch.zeros(items, dim, dtype=torch.bfloat16, device=DEV)
    keep = torch.cat([torch.arange(40), torch.arange(items - 61, items)]).to(DEV)
    rows = randn(keep.numel(), dim, seed=17, dtype=torch.bfloat16)
    table[keep] = rows
    bias = torch.full((items,), -math.inf, device=DEV)
    bias[keep] = 0.0
    x = randn(37, dim, seed=18, dtype=torch.bfloat16)
    pick = torch.randint(0, keep.numel(), (37,), generator=torch.Generator().manual_seed(19)).to(DEV)
    grad = torch.ones(37, device=DEV)
    loss, lse = ops.softmax_loss_forward(x, table, keep[pick], bias, 0.1)
    dx, dt = ops.softmax_loss_backward(grad, x, table, keep[pick], lse, bias, 0.1, [True, True])
    want = plain.softmax_loss(x, rows, pick, None, 0.1, grad)
    plain.close(loss, want[0])
    plain.close(dx, want[1])
    plain.close(dt[keep], want[2])
    assert not dt[1000:items - 1000:1000].any()


# ---- streams, graphs, workspaces -------------------------------------------------------------------------------------

def head_step(ops, x, weight, bias, table, target, gloss):
    """Forward and backward of the head, pass by pass."""
    a = ops.dropout(x, 0.2, 5, 1)
    y, mean, rstd = ops.layer_norm_forward(a, weight, bias, 1e-5)
    loss, lse = ops.softmax_loss_forward(y, table, target, None, 0.3)
    dy, dt = ops.softmax_loss_backward(gloss, y, table, target, lse, None, 0.3, [True, True])
    da, dw, db = ops.layer_norm_backward(dy, a, weight, mean, rstd, [True, True, True])
    return loss, ops.dropout(da, 0.2, 5, 1), dw, db, dt


def test_head_captured_and_replayed(ops):
    x, table, target, gloss = loss_case(300, 1500, 64, "bf16", 21)
    weight, bias = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    head_step(ops, x, weight, bias, table, target, gloss)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):   # two graphs side by side: each has its own workspaces
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(head_step(ops, x, weight, bias, table, target, gloss))
        graphs.append(graph)
    for k in range(3):
        x.copy_(randn(300, 64, seed=30 + k, dtype=torch.bfloat16))
        target.copy_(torch.randint(0, 1500, (300,), generator=torch.Generator().manual_seed(k)))
        want = head_step(ops, x, weight, bias, table, target, gloss)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_head_captured_with_autograd(ops):
    x, table, target, gloss = loss_case(100, 400, 64, "f32", 22)
    table.requires_grad_()

    def step():
        loss = ops.softmax_loss(ops.layer_norm(x, None, None), table, target, None, 0.3)
        return loss.detach(), torch.autograd.grad(loss, (table,), gloss)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        x.copy_(randn(100, 64, seed=40 + k))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_head_graph_holds_kernels_only():
    L = capi.lib()
    x, table, target, gloss = loss_case(100, 401, 20, "f32", 23)   # 20 columns of float32; odd item count
    loss, lse = torch.empty(100, device=DEV), torch.empty(100, device=DEV)
    dx, dt = torch.empty_like(x), torch.empty_like(table)
    dw, db, y = torch.empty(20, device=DEV), torch.empty(20, device=DEV), torch.empty_like(x)
    f, b, n = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
    capi.check(L.recsdk_softmax_loss_workspace(100, 401, 20, capi.DT_F32, 20, 20, f, b))
    capi.check(L.recsdk_layer_norm_workspace(100, 20, n))
    ws = torch.empty(max(f.value, b.value, n.value), dtype=torch.uint8, device=DEV)
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        s = host._stream()
        p = lambda t: t.data_ptr()  # noqa: E731
        capi.check(L.recsdk_layer_norm_forward(p(x), 100, 20, 20, capi.DT_F32, None, None, capi.DT_F32, 1e-5, p(y), p(loss), p(lse), s))
        capi.check(L.recsdk_layer_norm_backward(p(y), p(x), 100, 20, 20, capi.DT_F32, None, capi.DT_F32, p(loss), p(lse), p(dx),
                                                p(dw), p(db), p(ws), ws.numel(), s))
        capi.check(L.recsdk_softmax_loss_forward(p(x), 100, 20, p(table), 401, 20, 20, capi.DT_F32, p(target), None, 0.5, p(loss),
                                                 p(lse), p(ws), ws.numel(), s))
        capi.check(L.recsdk_softmax_loss_backward(p(gloss), p(x), 100, 20, p(table), 401, 20, 20, capi.DT_F32, p(target), None, 0.5,
                                                  p(lse), p(dx), p(dt), p(ws), ws.numel(), s))
    assert set(host.graph_node_kinds(graph.raw_cuda_graph())) == {"kernel"}


def test_head_on_two_streams_at_once(ops):
    cases = [loss_case(200 + 50 * k, 3000, 64, "bf16", 50 + k) for k in range(2)]
    weight, bias = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    want = [head_step(ops, x, weight, bias, table, target, g) for x, table, target, g in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for s, (x, table, target, g) in zip(streams, cases):
        with torch.cuda.stream(s):
            got.append([head_step(ops, x, weight, bias, table, target, g) for _ in range(5)][-1])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_outputs_are_written_whole_and_nothing_behind_them():
    L = capi.lib()
    x, table, target, gloss = loss_case(33, 130, 36, "f32", 24)
    f, b = ctypes.c_int64(), ctypes.c_int64()
    capi.check(L.recsdk_softmax_loss_workspace(33, 130, 36, capi.DT_F32, 36, 36, f, b))
    # each buffer with a margin behind it that has to stay as it is
    def room(n):
        return torch.full((n + 64,), 777.0, device=DEV)

    loss, lse, dx, dt = room(33), room(33), room(33 * 36), room(130 * 36)
    wf, wb = room(f.value // 4), room(b.value // 4)
    s = host._stream()
    capi.check(L.recsdk_softmax_loss_forward(x.data_ptr(), 33, 36, table.data_ptr(), 130, 36, 36, capi.DT_F32, target.data_ptr(), None,
                                             0.5, loss.data_ptr(), lse.data_ptr(), wf.data_ptr(), f.value, s))
    capi.check(L.recsdk_softmax_loss_backward(gloss.data_ptr(), x.data_ptr(), 33, 36, table.data_ptr(), 130, 36, 36, capi.DT_F32,
                                              target.data_ptr(), None, 0.5, lse.data_ptr(), dx.data_ptr(), dt.data_ptr(),
                                              wb.data_ptr(), b.value, s))
    want = plain.softmax_loss(x, table, target, None, 0.5, gloss)
    plain.close(loss[:33], want[0])
    plain.close(dx[:33 * 36].reshape(33, 36), want[1])
    plain.close(dt[:130 * 36].reshape(130, 36), want[2])
    for t, n in ((loss, 33), (lse, 33), (dx, 33 * 36), (dt, 130 * 36), (wf, f.value // 4), (wb, b.value // 4)):
        assert (t[n:] == 777.0).all()


# ---- the head behind the lookup, as it is used -----------------------------------------------------------------------

def test_lookup_dropout_norm_loss_and_table_update(ops):
    """Pooled lookup -> dropout -> layer norm -> softmax loss over an item table, and the gradient back through the lookup's
    fused SGD update: one training step against the same step in 64 bits."""
    rows, dim, batch, items, lr = 500, 64, 96, 700, 0.1
    g = torch.Generator().manual_seed(60)
    emb = torch.randn(rows, dim, generator=g)
    lengths = torch.randint(1, 6, (batch,), generator=g)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), lengths.cumsum(0)])
    indices = torch.randint(0, rows, (int(offsets[-1]),), generator=g)
    x0, table, target, gloss = loss_case(batch, items, dim, "f32", 61)
    weight, bias = 1 + 0.1 * randn(dim, seed=62), randn(dim, seed=63, std=0.1)

    dev = emb.reshape(-1).to(DEV)
    none = torch.empty(0, device=DEV)
    w_off = torch.zeros(1, dtype=torch.long, device=DEV)
    d_off = torch.tensor([0, dim], dtype=torch.int32, device=DEV)
    hcs = torch.tensor([0, rows], dtype=torch.long, device=DEV)
    leaf = torch.zeros(1, device=DEV, requires_grad=True)
    pooled = torch.ops.fbgemm.split_embedding_codegen_lookup_sgd_function(
        leaf, dev, none, none, none, w_off, d_off, dim, dim, hcs, 10, indices.to(DEV), offsets.to(DEV), capi.POOL_SUM, None, None,
        none, False, 0.0, False, learning_rate=lr)
    leaves = [t.detach().requires_grad_() for t in (weight, bias, table)]
    loss = ops.softmax_loss(ops.layer_norm(ops.dropout(pooled, 0.2, 5, 1), leaves[0], leaves[1]), leaves[2], target, None, 0.3)
    (loss * gloss).sum().backward()

    e = emb.double().requires_grad_()
    p64 = torch.stack([e[indices[offsets[k]:offsets[k + 1]]].sum(0) for k in range(batch)])
    keep = plain.dropout(pooled, 0.2, 5, 1)[1].double() * (65536 / round(65536 * 0.8))
    w64, b64, t64 = (t.detach().double().cpu().requires_grad_() for t in leaves)
    a = p64 * keep
    hat = (a - a.mean(1, keepdim=True)) / torch.sqrt(a.var(1, unbiased=False, keepdim=True) + 1e-5)
    z = 0.3 * (hat * w64 + b64) @ t64.T
    l64 = torch.logsumexp(z, 1) - z.gather(1, target.cpu()[:, None])[:, 0]
    (l64 * gloss.double().cpu()).sum().backward()
    # float32 throughout: sums of at most 700 terms, each step's relative error well below 1e-5 of the largest value
    for got, want in ((loss, l64), (leaves[0].grad, w64.grad), (leaves[1].grad, b64.grad), (leaves[2].grad, t64.grad),
                      (dev.reshape(rows, dim), emb.double() - lr * e.grad)):
        want = want.detach()
        assert (got.detach().double().cpu() - want).abs().max() <= 2e-5 * want.abs().max()


def test_head_configuration_of_the_benchmark_runs(capsys):
    import json

    from recsdk_amd import config_bench as cb
    from recsdk_amd import synth

    cb.run_head(cb.default_args(config="head", steps=2, warmup=1), torch, capi, host, synth)
    lines = [json.loads(text) for text in capsys.readouterr().out.splitlines() if text.startswith("{")]
    assert len(lines) == 2 and all(d["config"] == "HEAD" and d["TFLOPs"] > 0 for d in lines)


@pytest.mark.parametrize("each", [1.015, 1.0, 0.6])
def test_bfloat16_gradients_are_off_by_their_own_rounding(ops, each):
    """Rows of equal weight, just above a power of two, where the rounding of the values would weigh most: the gradients' error
    stays near what rounding the exact gradients alone leaves."""
    x, table, target, _ = loss_case(256, 20000, 64, "bf16", 81)
    grad = torch.full((256,), each / 256, device=DEV)
    leaves = [t.detach().requires_grad_() for t in (x, table)]
    got = torch.autograd.grad(ops.softmax_loss(*leaves, target, None, 0.3), leaves, grad)
    z = 0.3 * x.double() @ table.double().t()
    q = torch.softmax(z, 1)
    q[torch.arange(256, device=DEV), target] -= 1
    q *= 0.3 * each / 256
    for a, exact in zip(got, (q @ table.double(), q.t() @ x.double())):
        own = (exact.bfloat16().double() - exact).norm()
        # beside the targets' terms (2^-16 after two rounds) the other probabilities, 2^-8 off at most, make up a few percent of
        # the gradients of x and less of the table's
        assert (a.double() - exact).norm() <= 1.15 * own


# ---- more rows than one launch has blocks for, rows far apart, gradients asked for one by one ---------------------------------

def test_layer_norm_more_wide_rows_than_blocks(ops):
    # rows off the 16-byte borders, with gaps, past what a block holds: a block per row, for 65536 of them at a time
    rows, dim = 65600, 4097
    wide = torch.randn(rows, dim + 2, generator=torch.Generator(DEV).manual_seed(90), device=DEV).bfloat16()
    x = wide[:, 1:dim + 1]
    weight = 1 + randn(dim, seed=91, std=0.1)
    bias = randn(dim, seed=92)
    grad = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
    grad[-100:] = randn(100, dim, seed=93, dtype=torch.bfloat16)
    y, mean, rstd = ops.layer_norm_forward(x, weight, bias)
    dx, dw, db = ops.layer_norm_backward(grad, x, weight, mean, rstd, [True, True, True])
    some = torch.cat([torch.arange(40), torch.arange(rows - 100, rows)]).to(DEV)
    want = plain.layer_norm(x[some], weight, bias, 1e-5, grad[some])
    plain.close(y[some], want[0], "y")
    plain.close(dx[some], want[1], "dx")
    plain.close(dw, want[2], "dweight")   # the other rows' gradients are zero
    plain.close(db, want[3], "dbias")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_softmax_loss_more_rows_than_blocks(ops, kind):
    x, table, target, grad = loss_case(525_000, 9, 5, kind, 94)   # padded rows, 65536 blocks of eight of them at a time
    check_loss(ops, x, table, target, None, 0.5, grad)


@pytest.mark.parametrize("kind,rows,items,dim", [("f32", 801, 33001, 200), ("bf16", 642, 65800, 250)])
def test_softmax_loss_last_items_in_pieces(ops, kind, rows, items, dim):
    # one round of blocks over the items and a few more blocks, which share out the rows of x
    x, table, target, grad = loss_case(rows, items, dim, kind, 99)
    target[::7] = torch.randint(items - 300, items, (target[::7].numel(),), generator=torch.Generator().manual_seed(100)).to(DEV)
    target[3] = -1
    check_loss(ops, x, table, target, None, 3 / math.sqrt(dim), grad)


def test_softmax_loss_large_table_and_no_rows(ops):
    x, table, target, grad = loss_case(4, 300_000, 256, "bf16", 95)
    torch.full_like(table, 7.0)   # what the gradient's memory may hold before
    _, dt = ops.softmax_loss_backward(grad[:0], x[:0], table, target[:0], grad[:0], None, 1.0, [False, True])
    assert not dt.any()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [8, 9, 10, 11, 12, 13, 14, 15, 31, 67, 125, 254])
def test_softmax_loss_rows_that_end_inside_a_piece(ops, kind, dim):
    # tables whose last row ends with the allocation, at each place in a 16-byte piece; strides of no whole pieces
    x, table, target, grad = loss_case(45, 130, dim, kind, 300 + dim)
    check_loss(ops, x, table, target, None, 3 / math.sqrt(dim), grad)
    wide = torch.full((130, dim + 3), math.nan, dtype=TYPES[kind], device=DEV)
    wide[:, :dim] = table
    check_loss(ops, x, wide[:, :dim], target, None, 3 / math.sqrt(dim), grad)   # what lies behind a row is not looked at
    few = torch.full((45, dim + 5), math.inf, dtype=TYPES[kind], device=DEV)
    few[:, :dim] = x
    check_loss(ops, few[:, :dim], table, target, None, 3 / math.sqrt(dim), grad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,items", [(1030, 140_000), (5000, 3000)])   # a table read as it lies, and one that is copied
def test_softmax_loss_rows_off_the_borders_are_read_as_padded_ones(ops, kind, rows, items):
    x, table, target, grad = loss_case(rows, items, 250, kind, 97)
    leaves = [t.detach().requires_grad_() for t in (x, table)]
    dx, dt = torch.autograd.grad(ops.softmax_loss(*leaves, target, None, 0.2), leaves, grad)
    padded = [torch.nn.functional.pad(t.detach(), (0, 6)).requires_grad_() for t in (x, table)]
    px, pt = torch.autograd.grad(ops.softmax_loss(*padded, target, None, 0.2), padded, grad)
    assert torch.equal(dx, px[:, :250]) and torch.equal(dt, pt[:, :250])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_softmax_loss_rows_far_apart(ops, kind):
    x, table, target, grad = loss_case(5, 9, 64, kind, 96)
    far = torch.zeros(9, 2 ** 22 + 8, dtype=TYPES[kind], device=DEV)
    far[:, :64] = table
    check_loss(ops, x, far[:, :64], target, None, 0.4, grad)
    far[:5, :64] = x
    check_loss(ops, far[:5, :64], table, target, None, 0.4, grad)


@pytest.mark.parametrize("weighted", [True, False])
def test_gradients_of_some_inputs_only(ops, weighted):
    x, weight, bias, grad = norm_case(70, 100, "f32", "f32", 97)
    leaves = [t.requires_grad_() for t in ((x, weight, bias) if weighted else (x, bias))]

    def layer(inputs):
        return ops.layer_norm(inputs[0], inputs[1] if weighted else None, inputs[-1])

    whole = torch.autograd.grad(layer(leaves), leaves, grad)
    for leaf, want in zip(leaves, whole):
        assert torch.equal(torch.autograd.grad(layer(leaves), (leaf,), grad)[0], want)
        only = [t if t is leaf else t.detach() for t in leaves]
        assert torch.equal(torch.autograd.grad(layer(only), (leaf,), grad)[0], want)
    x, table, target, grad = loss_case(70, 300, 64, "bf16", 98)
    leaves = [x.requires_grad_(), table.requires_grad_()]
    whole = torch.autograd.grad(ops.softmax_loss(*leaves, target), leaves, grad)
    for leaf, want in zip(leaves, whole):
        assert torch.equal(torch.autograd.grad(ops.softmax_loss(*leaves, target), (leaf,), grad)[0], want)


# ---- refusals that need a device -------------------------------------------------------------------------------------

def test_refusals_of_the_torch_operators(ops):
    x, table, target, grad = loss_case(10, 30, 16, "f32", 70)
    ok = dict(match="recsdk::")
    for bad in (lambda: ops.softmax_loss(x, table.bfloat16(), target), lambda: ops.softmax_loss(x.half(), table.half(), target),
                lambda: ops.softmax_loss(x, table[:, :8], target), lambda: ops.softmax_loss(x, table, target[:5]),
                lambda: ops.softmax_loss(x, table, target.float()), lambda: ops.softmax_loss(x, table[:0], target),
                lambda: ops.softmax_loss(x, table, target, torch.zeros(29, device=DEV)),
                lambda: ops.softmax_loss(x, table, target, torch.zeros(30, device=DEV, dtype=torch.float64)),
                lambda: ops.softmax_loss(x, table, target, torch.zeros(30, device=DEV, requires_grad=True)),
                lambda: ops.softmax_loss(x, table.cpu(), target), lambda: ops.softmax_loss(x, table, target.cpu()),
                lambda: ops.softmax_loss(randn(4, 257), randn(5, 257), target[:4]), lambda: ops.softmax_loss(x[0], table, target[:1]),
                lambda: ops.layer_norm(x, torch.ones(15, device=DEV)), lambda: ops.layer_norm(x, torch.ones(16, device=DEV).half()),
                lambda: ops.layer_norm(x, torch.ones(16)), lambda: ops.layer_norm(x.int()), lambda: ops.layer_norm(x, None, None, -1.0),
                lambda: ops.layer_norm(x, torch.ones(16, device=DEV), torch.ones(16, device=DEV).bfloat16()),
                lambda: ops.dropout(x, -0.1, 0), lambda: ops.dropout(x, 1.5, 0), lambda: ops.dropout(x, math.nan, 0),
                lambda: ops.dropout(x.long(), 0.5, 0), lambda: ops.dropout(x, 0.5, 0, 0, torch.zeros(2, dtype=torch.long, device=DEV)),
                lambda: ops.dropout(x, 0.5, 0, 0, torch.zeros(1, dtype=torch.long))):
        with pytest.raises(RuntimeError, **ok):
            bad()
    loss, lse = ops.softmax_loss_forward(x, table, target)
    for bad in (lambda: ops.softmax_loss_backward(grad[:5], x, table, target, lse, None, 1.0, [True, True]),
                lambda: ops.softmax_loss_backward(grad.double(), x, table, target, lse, None, 1.0, [True, True])):
        with pytest.raises(RuntimeError, **ok):
            bad()
    leaf = x.detach().requires_grad_()
    for y in (ops.dropout(leaf, 0.5, 1), ops.layer_norm(leaf), ops.softmax_loss(leaf, table, target)):
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(y.sum(), (leaf,), create_graph=True)


def test_a_short_workspace_is_refused():
    L = capi.lib()
    x, table, target, gloss = loss_case(100, 400, 64, "f32", 71)
    f, b, n = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
    capi.check(L.recsdk_softmax_loss_workspace(100, 400, 64, capi.DT_F32, 64, 64, f, b))
    capi.check(L.recsdk_layer_norm_workspace(100, 64, n))
    out = torch.full((400 * 64,), 777.0, device=DEV)
    args = (x.data_ptr(), 100, 64, table.data_ptr(), 400, 64, 64, capi.DT_F32, target.data_ptr(), None, 0.5)
    s = host._stream()
    assert L.recsdk_softmax_loss_forward(*args, out.data_ptr(), out.data_ptr(), out.data_ptr(), f.value - 1, s) == capi.ECAPACITY
    assert L.recsdk_softmax_loss_backward(gloss.data_ptr(), *args, gloss.data_ptr(), out.data_ptr(), out.data_ptr(), out.data_ptr(),
                                          b.value - 1, s) == capi.ECAPACITY
    assert L.recsdk_layer_norm_backward(x.data_ptr(), x.data_ptr(), 100, 64, 64, capi.DT_F32, None, capi.DT_F32, gloss.data_ptr(),
                                        gloss.data_ptr(), out.data_ptr(), out.data_ptr(), None, out.data_ptr(), n.value - 1, s) == capi.ECAPACITY
    torch.cuda.synchronize()
    assert (out == 777.0).all()

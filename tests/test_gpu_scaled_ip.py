"""InnerProduct of 8-bit operands with block scales, against its definition in 64 bits."""
import math

import pytest
import torch

from block8_util import DEV, TYPES, ULP, matrix, quantized, round_room, widen

pytestmark = pytest.mark.gpu


def operands(rows, inputs, outputs, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, inputs, device=DEV, generator=g)
    x[:, torch.randint(0, inputs, (1 + inputs // 200,), device=DEV, generator=g)] *= 30
    w = torch.randn(outputs, inputs, device=DEV, generator=g) * inputs ** -0.5
    return quantized(x, 1) + quantized(w, 128)


def wanted(x, xs, w, ws, bias=None):
    """The product in 64 bits, and the sum of the magnitudes of its terms."""
    a = x.double() * widen(xs.t(), 1, x.shape).double()
    b = w.double() * widen(ws, 128, w.shape).double()
    y, size = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def room(size, inputs):
    """fp32 sums: the tensor core adds the 128 products of a block, each exact, with at most 128 roundings (or truncations: 2 halves) of partial
    sums; two scale products, and a sum over the blocks and parts.  Partial sums are no larger than the sum of magnitudes."""
    return size * (2 * 128 + 4 + -(-inputs // 128) + 8) * ULP


ACT = {"identity": lambda v: v, "relu": torch.relu, "relu6": lambda v: v.clamp(0, 6), "sigmoid": torch.sigmoid, "tanh": torch.tanh}


def run(x, xs, w, ws, out="fp32", bias=None, act="identity", extra=0, shift=0, stream=None):
    from dlprimitives_b200 import capi
    y, memory = matrix(x.shape[0], w.shape[0], TYPES[out], extra, shift)
    memory.fill_(-77)
    capi.scaled_inner_product(x, xs, w, ws, y, bias=bias, activation=act, stream=stream)
    got = y.clone()
    assert capi.device_status() == 0
    y.fill_(-77)
    assert bool((memory == -77).all())              # rows behind the last and columns behind a row's end are as they were
    return got


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 65, 100, 128, 129, 256, 300])
@pytest.mark.parametrize("inputs,outputs", [(128, 128), (1000, 300), (16, 1), (4096, 520), (129, 2000)])
def test_sizes(rows, inputs, outputs):
    x, xs, w, ws = operands(rows, inputs, outputs, rows + inputs)
    y, size = wanted(x, xs, w, ws)
    got = run(x, xs, w, ws)
    assert bool(((got.double() - y).abs() <= room(size, inputs)).all()), float(((got.double() - y).abs() / room(size, inputs)).max())


@pytest.mark.parametrize("rows,inputs,outputs", [(1, 1, 1), (1, 17, 3), (5, 127, 129), (700, 2500, 1111), (1, 16384, 4096), (3, 16383, 129),
                                                (1025, 260, 257), (2048, 512, 640)])
def test_more_sizes(rows, inputs, outputs):
    x, xs, w, ws = operands(rows, inputs, outputs, rows)
    y, size = wanted(x, xs, w, ws)
    got = run(x, xs, w, ws)
    assert bool(((got.double() - y).abs() <= room(size, inputs)).all())


@pytest.mark.parametrize("rows", [1, 20, 48, 200, 513])
@pytest.mark.parametrize("out", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("act", ["identity", "relu", "relu6", "sigmoid", "tanh"])
def test_types_bias_activation(rows, out, act):
    x, xs, w, ws = operands(rows, 600, 333, rows)
    bias = torch.randn(333, device=DEV)
    y, size = wanted(x, xs, w, ws, bias)
    for extra, shift in ((0, 0), (3, 0), (19, 16), (7, 1)):
        got = run(x, xs, w, ws, out, bias, act, extra, shift)
        # the activations are no steeper than 1; tanhf and expf are within 2 units
        want = ACT[act](y)
        assert bool(((got.double() - want).abs() <= room(size, 600) + 8 * ULP + round_room(want, got.dtype) * (1 + 2.0 ** -8)).all())


def test_rows_of_operands_far_apart():
    """Strides other than the lengths, of all that has one."""
    rows, inputs, outputs = 150, 300, 260
    x, xs, w, ws = operands(rows, inputs, outputs, 1)
    y, size = wanted(x, xs, w, ws)
    far_x, _ = matrix(rows, inputs, TYPES["e4m3"], 4096 - inputs, 32)
    far_w, _ = matrix(outputs, inputs, TYPES["e4m3"], 512 - inputs, 16)
    far_x.copy_(x)
    far_w.copy_(w)
    far_xs = torch.full((3, 999), math.nan, device=DEV)[:, 1:rows + 1]
    far_ws = torch.full((3, 17), math.nan, device=DEV)[:, 2:5]
    far_xs.copy_(xs)
    far_ws.copy_(ws)
    for n in (150, 40):
        got = run(far_x[:n], far_xs[:, :n], far_w, far_ws, "fp32", None, "identity", 5)
        assert bool(((got.double() - y[:n]).abs() <= room(size, inputs)[:n]).all())


@pytest.mark.parametrize("rows", [3, 300])
def test_padding_is_not_read(rows):
    """NaN numbers in the columns between a row's end and the next row, and in rows behind the last."""
    inputs, outputs = 200, 100
    x, xs, w, ws = operands(rows, inputs, outputs, 3)
    y, size = wanted(x, xs, w, ws)
    big_x = torch.full((rows + 130, 208), 0x7f, dtype=torch.uint8, device=DEV).view(TYPES["e4m3"])
    big_w = torch.full((outputs + 130, 208), 0x7f, dtype=torch.uint8, device=DEV).view(TYPES["e4m3"])
    big_x[:rows, :inputs] = x
    big_w[:outputs, :inputs] = w
    got = run(big_x[:rows, :inputs], xs, big_w[:outputs, :inputs], ws)
    assert bool(((got.double() - y).abs() <= room(size, inputs)).all())


@pytest.mark.parametrize("rows", [5, 200])
def test_what_is_not_finite_stays_in_its_row(rows):
    x, xs, w, ws = operands(rows, 512, 256, 7)
    xs[1, 2] = math.nan
    xs[0, 3] = math.inf
    x.view(torch.uint8)[4, 300] = 0x7f
    y, _ = wanted(x, xs, w, ws)
    got = run(x, xs, w, ws)
    bad = torch.zeros(rows, dtype=torch.bool, device=DEV)
    bad[2:5] = True
    assert bool(got[~bad].isfinite().all())
    assert bool(got[2].isnan().all()) and bool(got[4].isnan().all()) and not bool(got[3].isfinite().any())
    relu = run(x, xs, w, ws, act="relu")
    assert bool((relu[2] == 0).all())               # relu makes a NaN 0, as everywhere in this library


@pytest.mark.parametrize("rows", [1, 48, 130, 600])
def test_same_bits_each_time(rows):
    x, xs, w, ws = operands(rows, 4100, 1500, 11)
    first = run(x, xs, w, ws)
    for _ in range(5):
        assert torch.equal(run(x, xs, w, ws), first)


@pytest.mark.parametrize("rows", [1, 24, 70, 400])
def test_captured_and_on_two_streams(rows):
    from dlprimitives_b200 import capi
    x, xs, w, ws = operands(rows, 1024, 900, 13)
    x2, xs2, _, _ = operands(rows, 1024, 900, 14)
    want, want2 = run(x, xs, w, ws), run(x2, xs2, w, ws)
    ys = [torch.empty_like(want) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, a, b, y in zip(streams, (x, x2), (xs, xs2), ys):
            capi.scaled_inner_product(a, b, w, ws, y, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(ys[0], want) and torch.equal(ys[1], want2)
    graph = torch.cuda.CUDAGraph()
    cx, cxs, y = x.clone(), xs.clone(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        for _ in range(3):
            capi.scaled_inner_product(cx, cxs, w, ws, y)
    for a, b, e in ((x2, xs2, want2), (x, xs, want)):
        cx.copy_(a)
        cxs.copy_(b)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, e)
    assert capi.device_status() == 0


def test_no_rows():
    from dlprimitives_b200 import capi
    x, xs, w, ws = operands(4, 256, 256, 1)
    y = torch.full((4, 256), 5.0, device=DEV)
    capi.scaled_inner_product(x[:0], xs[:, :0], w, ws, y[:0])
    torch.cuda.synchronize()
    assert bool((y == 5).all())

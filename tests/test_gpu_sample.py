"""Draw of a class from logits, against its definition in 64 bits: the same class in every row."""
import math

import pytest
import torch

from block8_util import DEV, TYPES

pytestmark = pytest.mark.gpu


def wanted(x, u, temperature=None, k=None, p=None, m=None):
    """Row by row on the CPU, in 64 bits, from the definition."""
    rows, n = x.shape
    x, u = x.double().cpu(), u.double().cpu()
    tokens = []
    for r in range(rows):
        t = 1.0 if temperature is None else float(temperature[r])
        z = torch.where(x[r].isnan(), -math.inf, x[r])
        top = float(z.max())
        if top == -math.inf:
            tokens.append(-1)
            continue
        if not t > 0:
            tokens.append(int((z == top).nonzero()[0]))
            continue
        w = torch.where(z == top, torch.ones_like(z), torch.exp((z - top) / t))
        w = torch.where(z == -math.inf, torch.zeros_like(w), w)
        order = torch.sort(z, descending=True, stable=True).indices
        count = n if k is None or not 0 < int(k[r]) < n else int(k[r])
        s = w[order][:count].cumsum(0)
        if p is not None and float(p[r]) < 1:
            count = min(count, 1 + int((s[:-1] < float(p[r]) * s[-1]).sum()))
        kept = torch.zeros(n, dtype=torch.bool)
        kept[order[:count]] = True
        if m is not None and float(m[r]) > 0:
            kept &= w >= min(1.0, float(m[r]))
        run = (w * kept).cumsum(0)
        tokens.append(int(((w * kept > 0) & (run > float(u[r]) * run[-1])).nonzero()[0]))
    return torch.tensor(tokens, dtype=torch.int32)


def run(x, u, **kw):
    from dlprimitives_b200 import capi
    memory = torch.full((x.shape[0] + 2,), 12345, dtype=torch.int32, device=DEV)
    capi.sample(x, u, memory[1:-1], **kw)
    assert capi.device_status() == 0
    assert int(memory[0]) == 12345 and int(memory[-1]) == 12345
    return memory[1:-1].cpu()


def draw(rows, n, kind, seed, spread=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = spread * torch.randn(rows, n, device=DEV, generator=g)
    x[torch.rand(rows, n, device=DEV, generator=g) < 0.02] = -math.inf
    return x.to(TYPES[kind]), torch.rand(rows, device=DEV, generator=g), g


def settings(rows, n, which, g):
    r = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, device=DEV, generator=g)       # noqa: E731
    kw = {}
    if "t" in which:
        kw["temperature"] = torch.where(r(0, 1) < 0.2, torch.zeros(rows, device=DEV), r(0.2, 2.0))
    if "k" in which:
        kw["top_k"] = torch.where(r(0, 1) < 0.2, torch.zeros(rows, device=DEV), r(1, min(n, 300))).int()
    if "p" in which:
        kw["top_p"] = torch.where(r(0, 1) < 0.2, torch.ones(rows, device=DEV), r(0.0, 1.0))
    if "m" in which:
        kw["min_p"] = torch.where(r(0, 1) < 0.2, torch.zeros(rows, device=DEV), r(0.0, 0.3))
    return kw


def check(x, u, kw):
    short = {"temperature": "temperature", "top_k": "k", "top_p": "p", "min_p": "m"}
    got, want = run(x, u, **kw), wanted(x, u, **{short[a]: b for a, b in kw.items()})
    assert torch.equal(got, want), (got[got != want], want[got != want])


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("which", ["", "t", "k", "p", "m", "tkpm"])
@pytest.mark.parametrize("rows,n", [(3, 1), (5, 2), (7, 33), (40, 1000), (9, 1025), (4, 32000), (3, 128000), (2, 262145)])
def test_against_the_definition(kind, which, rows, n):
    x, u, g = draw(rows, n, kind, rows * n)
    check(x, u, settings(rows, n, which, g))


@pytest.mark.parametrize("rows", [1, 2, 37, 150, 400])
def test_row_counts(rows):
    x, u, g = draw(rows, 5003, "fp32", rows)
    check(x, u, settings(rows, 5003, "tkp", g))


@pytest.mark.parametrize("n", [100, 5000, 131072])
@pytest.mark.parametrize("which", ["k", "p", "kp", "m"])
def test_equal_logits(n, which):
    """A few different values, each many times: which of the equal ones are kept goes by index."""
    g = torch.Generator(device=DEV).manual_seed(n)
    x = torch.randint(0, 3, (6, n), device=DEV, generator=g).float()
    x[4] = 0.25                                     # a row of one value
    x[5] = -0.0                                     # zeros of both signs are equal
    x[5, ::2] = 0.0
    check(x, torch.rand(6, device=DEV, generator=g), settings(6, n, which, g))


def test_random_numbers_over_the_whole_range():
    """u from 0 to the last number below 1: the first and the last class that is kept; each class as often as its mass says."""
    n = 4096
    u = torch.cat([torch.tensor([0.0, 2.0 ** -149, 1 - 2.0 ** -24], device=DEV), (torch.arange(n, device=DEV) + 0.5) / n])
    x = torch.full((len(u), 300), -math.inf, device=DEV)
    x[:, 10] = math.log(1.0)
    x[:, 100] = math.log(2.0)
    x[:, 299] = math.log(5.0)
    got = run(x, u)
    assert torch.equal(got[:3], torch.tensor([10, 10, 299], dtype=torch.int32))
    counts = torch.bincount(got[3:].long(), minlength=300)
    assert [int(counts[i]) for i in (10, 100, 299)] == [n // 8, n // 4, n - n // 8 - n // 4]
    check(x, u, {})


def test_masked_and_special_rows():
    low = torch.finfo(torch.float32).min
    x = torch.full((10, 2000), -math.inf, device=DEV)
    x[1, 1999] = -3.0                               # a single class is left
    x[2] = low                                      # masks of the type's lowest value: nothing is larger, so all are equal
    x[3] = low
    x[3, 7] = 1.0
    x[4, 5] = math.nan
    x[5, 5] = math.nan
    x[5, 6] = 2.0
    x[6, 100:] = 0.0
    x[6, 50] = x[6, 1500] = math.inf                # share all the mass
    x[7] = 1e38
    x[7, 3] = 3e38
    x[8, :4] = 80.0
    x[9] = -200.0
    for kw in ({}, {"top_p": torch.full((10,), 0.9, device=DEV)}, {"top_k": torch.full((10,), 3, dtype=torch.int32, device=DEV)},
               {"temperature": torch.zeros(10, device=DEV)}, {"min_p": torch.full((10,), 0.5, device=DEV)}):
        for v in (0.0, 0.4, 0.99):
            u = torch.full((10,), v, device=DEV)
            check(x, u, kw)
            got = run(x, u, **kw)
            assert int(got[0]) == -1 and int(got[4]) == -1 and int(got[1]) == 1999 and int(got[5]) == 6 and int(got[6]) in (50, 1500)
    check(x.half().float().half(), torch.full((10,), 0.7, device=DEV), {})


def test_settings_at_their_ends():
    n = 1000
    x, _, _ = draw(8, n, "fp32", 3)
    x[0, 3] = x[0, 500] = 50.0
    u = torch.full((8,), 0.999, device=DEV)
    f = lambda *v: torch.tensor(v, device=DEV)      # noqa: E731
    for kw in ({"top_p": f(0.0, -1.0, 1e-30, 0.5, 1.0, 2.0, math.nan, 1 - 2.0 ** -24)}, {"min_p": f(0.0, -1.0, 1.0, 5.0, 1e-30, 1e-9, 0.999, 0.5)},
               {"top_k": f(0, -5, 1, 2, n - 1, n, n + 1, 2 ** 31 - 1).int()}, {"temperature": f(0.0, -1.0, 1e-30, 1e-3, 1e3, 1e30, 0.01, 100.0)}):
        check(x, u, kw)


@pytest.mark.parametrize("top,t,m", [(0.0, 1.0, 0.25), (3.3, 0.7, 0.05), (math.log(8.0), 1.0, 0.125), (-1000.5, 2.0, 0.9), (1e30, 1.0, 0.5),
                                     (0.25, 1e-3, 1e-30), (2.0, 1e30, 0.5), (1.0, 1.0, 1.0), (0.0, 1.0, 1e-45)])
@pytest.mark.parametrize("n", [40, 5003, 40000])
def test_the_border_of_min_p(top, t, m, n):
    # One class beside the largest, a few fp32 numbers around the border (these are 2^-24 of the border apart, an exponential in 64 bits is
    # right to 2^-52), and far from it; u is near 1, so that the class drawn is the last one kept with a mass worth mentioning.
    top, m = float(torch.tensor(top)), float(torch.tensor(m))
    near = [torch.tensor(top + t * math.log(m), dtype=torch.float32).clamp(-3e38, top)]
    for up in (math.inf, -math.inf):
        v = near[0]
        for _ in range(40):
            v = torch.nextafter(v, torch.tensor(up))
            near.append(v)
    far = [top - 1e-6, top - 1.0, top - 50.0 * t, -3e38, 0.0, 1e-30, -1e-30]
    second = torch.tensor([min(float(v), top) for v in near + far if math.isfinite(v)], dtype=torch.float32)
    x = torch.full((len(second), n), -math.inf, device=DEV)
    x[:, 0], x[:, n - 1] = top, second.to(DEV)
    rows = len(second)
    u = torch.full((rows,), 1 - 2.0 ** -24, device=DEV)
    check(x, u, {"temperature": torch.full((rows,), t, device=DEV), "min_p": torch.full((rows,), m, device=DEV)})


def test_rows_far_apart_and_off_boundaries():
    memory = torch.full((7 * 9001 + 5,), math.inf, device=DEV)
    for shift in (0, 1, 3):
        x = memory[shift:shift + 7 * 9001].view(7, 9001)[:, :8190]
        src, u, g = draw(7, 8190, "fp32", shift)
        memory.fill_(math.inf)                       # what is no logit would win
        x.copy_(src)
        check(x, u, settings(7, 8190, "tkp", g))


@pytest.mark.parametrize("rows", [1, 200])
def test_captured_on_another_stream(rows):
    from dlprimitives_b200 import capi
    x, u, g = draw(rows, 30000, "bf16", rows)
    kw = settings(rows, 30000, "tkp", g)
    want = run(x, u, **kw)
    tokens, cu = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.zeros_like(u)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        for _ in range(2):
            capi.sample(x, cu, tokens, stream=s, **kw)
    cu.copy_(u)
    for _ in range(3):
        tokens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens.cpu(), want)


def test_no_rows():
    from dlprimitives_b200 import capi
    capi.sample(torch.empty(0, 100, device=DEV), torch.empty(0, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV))

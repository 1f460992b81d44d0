"""The operators with typed operands in a run, as a decoder's feed-forward layer and its head use them: norm with residual and 8-bit output, product,
gated quantisation, product, norm, product, draw.  Each step is held to its definition in 64 bits on what the step before it gave; eagerly, on
another stream, and captured."""
import pytest
import torch

from block8_util import DEV, TYPES, ULP, check_8_bits, quantized, widen

pytestmark = pytest.mark.gpu

HIDDEN, INNER, CLASSES = 640, 1416, 5003


class Layer:
    """Weights in bf16, brought into 8 bits by the library; buffers for `rows` rows."""

    def __init__(self, rows, seed):
        from dlprimitives_b200 import capi
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = lambda *shape: torch.randn(*shape, device=DEV, generator=g)         # noqa: E731
        self.rows = rows
        self.weights = {}
        for name, n, k in (("gate_up", 2 * INNER, HIDDEN), ("down", HIDDEN, INNER), ("head", CLASSES, HIDDEN)):
            w = (r(n, k) * k ** -0.5).bfloat16()
            q = self.eight(n, k)
            s = torch.empty(-(-n // 128), -(-k // 128), device=DEV)
            capi.quantize(w, q, s, block_rows=128)
            self.weights[name] = (w, q, s)
        self.norm1, self.norm2 = ((1 + 0.1 * r(HIDDEN)).bfloat16() for _ in range(2))
        self.x, self.residual = r(rows, HIDDEN).bfloat16(), (3 * r(rows, HIDDEN)).bfloat16()
        self.u, self.temperature = torch.rand(rows, device=DEV, generator=g), 0.5 + torch.rand(rows, device=DEV, generator=g)
        self.k, self.p = torch.full((rows,), 40, dtype=torch.int32, device=DEV), torch.full((rows,), 0.9, device=DEV)
        b = lambda *shape: torch.empty(*shape, dtype=torch.bfloat16, device=DEV)  # noqa: E731
        self.total1, self.total2, self.pair, self.out = b(rows, HIDDEN), b(rows, HIDDEN), b(rows, 2 * INNER), b(rows, HIDDEN)
        self.q1, self.q2, self.q3 = self.eight(rows, HIDDEN), self.eight(rows, INNER), self.eight(rows, HIDDEN)
        self.s1, self.s2, self.s3 = (torch.empty(-(-k // 128), rows, device=DEV) for k in (HIDDEN, INNER, HIDDEN))
        self.logits = torch.empty(rows, CLASSES, device=DEV)
        self.tokens = torch.empty(rows, dtype=torch.int32, device=DEV)

    @staticmethod
    def eight(n, k):
        return torch.empty(n, -(-k // 16) * 16, dtype=TYPES["e4m3"], device=DEV)[:, :k]

    def run(self, stream=None):
        from dlprimitives_b200 import capi
        w = {n: v[1:] for n, v in self.weights.items()}
        capi.rms_norm(self.x, self.norm1, self.q1, residual=self.residual, total=self.total1, scales=self.s1, stream=stream)
        capi.scaled_inner_product(self.q1, self.s1, *w["gate_up"], self.pair, stream=stream)
        capi.quantize(self.pair, self.q2, self.s2, gate="silu", stream=stream)
        capi.scaled_inner_product(self.q2, self.s2, *w["down"], self.out, stream=stream)
        capi.rms_norm(self.out, self.norm2, self.q3, residual=self.total1, total=self.total2, scales=self.s3, stream=stream)
        capi.scaled_inner_product(self.q3, self.s3, *w["head"], self.logits, stream=stream)
        capi.sample(self.logits, self.u, self.tokens, temperature=self.temperature, top_k=self.k, top_p=self.p, stream=stream)

    def results(self):
        return [t.clone() for t in (self.total1, self.q1, self.s1, self.pair, self.q2, self.s2, self.out, self.total2, self.q3, self.s3, self.logits, self.tokens)]


def product(q, s, w):
    a = q.double() * widen(s.t(), 1, q.shape).double()
    b = w[1].double() * widen(w[2], 128, w[1].shape).double()
    # as in test_gpu_scaled_ip.py: the roundings of 128-term sums and of the sum over blocks, of the terms' magnitudes
    return a @ b.t(), (a.abs() @ b.abs().t()) * (2 * 128 + 12 + -(-q.shape[1] // 128)) * ULP


@pytest.mark.parametrize("rows", [1, 7, 70, 300])
def test_each_step(rows):
    from dlprimitives_b200 import capi
    L = Layer(rows, rows)
    L.run()
    assert capi.device_status() == 0
    for _, q, s in L.weights.values():
        assert bool(q.float().isfinite().all()) and bool((s > 0).all())
    check_8_bits(L.weights["down"][1], L.weights["down"][2], L.weights["down"][0].double(), 128, 0.0)
    half = 2.0 ** -9                                 # bf16
    for x, r, w, q, s, total in ((L.x, L.residual, L.norm1, L.q1, L.s1, L.total1), (L.out, L.total1, L.norm2, L.q3, L.s3, L.total2)):
        h = x.double() + r.double()
        v = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * w.double()
        assert bool(((total.double() - h).abs() <= h.abs() * (2 * half)).all())
        check_8_bits(q, s.t(), v, 1, 40 * ULP)
    for q, s, w, y in ((L.q1, L.s1, "gate_up", L.pair), (L.q2, L.s2, "down", L.out), (L.q3, L.s3, "head", L.logits)):
        want, room = product(q, s, L.weights[w])
        assert bool(((y.double() - want).abs() <= room + (want.abs() * 2 * half if y.dtype == torch.bfloat16 else 0)).all()), w
    a, b = L.pair[:, :INNER].double(), L.pair[:, INNER:].double()
    check_8_bits(L.q2, L.s2.t(), a * torch.sigmoid(a) * b, 1, 10 * ULP)
    from test_gpu_sample import wanted
    assert torch.equal(L.tokens.cpu(), wanted(L.logits, L.u, L.temperature, L.k, L.p))
    # and all of it is near what the layer gives without 8 bits: two quantisations with steps of up to an eighth, whose errors (uniform, an eighth /
    # sqrt(12) of a value at the worst) the products average: well under a tenth in the norm
    w = {n: v[0].double() for n, v in L.weights.items()}
    h = L.x.double() + L.residual.double()
    v = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * L.norm1.double()
    pair = v @ w["gate_up"].t()
    out = (pair[:, :INNER] * torch.sigmoid(pair[:, :INNER]) * pair[:, INNER:]) @ w["down"].t()
    assert float((L.out.double() - out).norm() / out.norm()) < 0.1


@pytest.mark.parametrize("rows", [1, 70, 300])
def test_captured_and_on_another_stream(rows):
    from dlprimitives_b200 import capi
    L = Layer(rows, 100 + rows)
    L.run()
    torch.cuda.synchronize()
    want = L.results()
    bits = lambda t: t.contiguous().view(torch.uint8)            # noqa: E731
    s = torch.cuda.Stream()
    for t in (L.q1, L.q2, L.q3):
        t.view(torch.uint8).zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        L.run(stream=s)
    s.synchronize()
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(L.results(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        L.run(stream=torch.cuda.current_stream())
        L.run(stream=torch.cuda.current_stream())
    x = L.x.clone()
    L.x.normal_()
    for _ in range(2):
        graph.replay()
    L.x.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(L.results(), want))
    assert capi.device_status() == 0


def test_two_at_once():
    """Two layers of different sizes, launch by launch in turn on two streams that nothing orders."""
    from dlprimitives_b200 import capi
    layers = [Layer(3, 1), Layer(150, 2)]
    want = []
    for L in layers:
        L.run()
        torch.cuda.synchronize()
        want.append(L.results())
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(20):
        for L, s in zip(layers, streams):
            L.run(stream=s)
    torch.cuda.synchronize()
    for L, w in zip(layers, want):
        assert all(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in zip(L.results(), w))
    assert capi.device_status() == 0


def test_the_products_take_their_routes():
    """Which kernel a product goes to, by its size."""
    from dlprimitives_b200 import capi
    seen = []
    for rows, inputs, outputs in ((1, 1024, 512), (20, 1024, 512), (60, 1024, 512), (200, 8192, 512), (400, 512, 20000), (1000, 4096, 8000)):
        x, xs = quantized(torch.randn(rows, inputs, device=DEV), 1)
        w, ws = quantized(torch.randn(outputs, inputs, device=DEV), 128)
        y = torch.empty(rows, outputs, device=DEV)
        capi.scaled_inner_product(x, xs, w, ws, y)
        seen.append(capi.last_route())
    # the last three: few output tiles with a long K, cut along it; many tiles of a short K; two rounds of the widest tiles against four of the narrower
    assert [r[:2] for r in seen] == [("scaled_few", 16), ("scaled_few", 32), ("scaled_few", 64), ("scaled_few", 64), ("scaled_pair", 128), ("scaled_pair", 256)]
    assert all(r[2] > 1 for r in seen[:4])
    assert capi.device_status() == 0

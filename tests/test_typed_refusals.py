"""What the operators with typed operands refuse, before anything reaches a device: calls of the C ABI with made-up addresses."""
import ctypes

import pytest

A = 1 << 20                                          # an address with every alignment


def status(name, args, **fields):
    from dlprimitives_b200 import capi
    call = getattr(capi, args)(**fields)
    return getattr(capi.lib(), name)(ctypes.byref(call), None), capi.lib().dlp_last_error().decode()


def refused(name, args, good, changes):
    from dlprimitives_b200 import capi
    for change in changes:
        assert set(change) <= set(good)
        st, msg = status(name, args, **{**good, **change})
        assert st == capi.INVALID_ARGUMENT, change
        assert msg.startswith("Failed "), msg
    assert getattr(capi.lib(), name)(None, None) == capi.INVALID_ARGUMENT


def test_rms_norm():
    good = dict(x=A, x_stride=64, residual=A, residual_stride=64, total=A, total_stride=64, weight=A, type=2, y=A, y_stride=64, y_type=3, scales=A,
                scale_stride=8, rows=8, cols=64, eps=1e-5)
    refused("dlp_rms_norm_fwd", "RmsNormArgs", good, [
        dict(x=None), dict(weight=None), dict(y=None), dict(scales=None), dict(y_type=2), dict(residual=None), dict(type=3), dict(type=-1), dict(y_type=4),
        dict(rows=-1), dict(cols=0), dict(x_stride=63), dict(residual_stride=63), dict(total_stride=0), dict(y_stride=-64),
        dict(cols=200, x_stride=200, residual_stride=200, total_stride=200, y_stride=200, scale_stride=7),
        dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=A + 1), dict(weight=A + 1), dict(total=A + 1),
        dict(scales=A + 2), dict(type=0, x=A + 2)])


def test_quantize():
    good = dict(x=A, x_stride=600, type=2, gate=1, q=A, q_stride=300, scales=A, scale_stride=8, block_rows=1, rows=8, cols=300)
    refused("dlp_quantize_fwd", "QuantizeArgs", good, [
        dict(x=None), dict(q=None), dict(scales=None), dict(type=3), dict(gate=3), dict(gate=-1), dict(block_rows=2), dict(block_rows=128),
        dict(x_stride=599), dict(q_stride=299), dict(scale_stride=7), dict(rows=-1), dict(cols=0), dict(x=A + 1), dict(scales=A + 1),
        dict(gate=0, block_rows=128, rows=129, scale_stride=2)])


def test_scaled_ip():
    good = dict(x=A, x_stride=304, x_scales=A, x_scale_stride=8, w=A, w_stride=304, w_scales=A, w_scale_stride=3, bias=None, y=A, y_stride=200, y_type=2,
                activation=0, rows=8, inputs=300, outputs=200)
    refused("dlp_scaled_ip_fwd", "ScaledIpArgs", good, [
        dict(x=None), dict(x_scales=None), dict(w=None), dict(w_scales=None), dict(y=None), dict(x_stride=288), dict(x_stride=301), dict(w_stride=303),
        dict(w_stride=288), dict(x=A + 8), dict(w=A + 4), dict(x_scale_stride=7), dict(w_scale_stride=2), dict(y_stride=199), dict(y_type=3),
        dict(y_type=-1), dict(activation=5), dict(activation=-1), dict(rows=-1), dict(inputs=0), dict(outputs=0), dict(bias=A + 2), dict(y=A + 1),
        dict(x_scales=A + 2), dict(x_stride=1 << 41), dict(w_stride=1 << 41)])


def test_sample():
    good = dict(logits=A, stride=100, type=0, rows=4, classes=100, u=A, tokens=A)
    refused("dlp_sample_fwd", "SampleArgs", {**good, "top_k": None, "temperature": None}, [
        dict(logits=None), dict(u=None), dict(tokens=None), dict(stride=99), dict(type=3), dict(rows=-1), dict(classes=0),
        dict(classes=(1 << 22) + 1, stride=1 << 23), dict(logits=A + 2), dict(u=A + 1), dict(top_k=A + 2), dict(tokens=A + 3), dict(temperature=A + 1)])


def test_nothing_to_do_needs_no_tensors():
    assert status("dlp_rms_norm_fwd", "RmsNormArgs", cols=8, eps=1e-5)[0] == 0
    assert status("dlp_quantize_fwd", "QuantizeArgs", cols=8, block_rows=1)[0] == 0
    assert status("dlp_scaled_ip_fwd", "ScaledIpArgs", inputs=16, outputs=8)[0] == 0
    assert status("dlp_sample_fwd", "SampleArgs", classes=8)[0] == 0


def test_structures_are_the_headers():
    """The binding's structures have the header's fields, in its order."""
    import os
    import re
    from dlprimitives_b200 import capi
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "dlp_cuda.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, cls in (("dlp_rms_norm_args", capi.RmsNormArgs), ("dlp_quantize_args", capi.QuantizeArgs), ("dlp_scaled_ip_args", capi.ScaledIpArgs),
                      ("dlp_sample_args", capi.SampleArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        fields = []
        for line in body.split(";"):
            line = line.strip()
            if line:
                kind = ctypes.c_void_p if "*" in line else {"long": ctypes.c_longlong, "int": ctypes.c_int, "float": ctypes.c_float}[line.split()[0]]
                fields += [(re.split(r"[\s*]+", n.strip())[-1], kind) for n in line.split(",")]
        assert fields == cls._fields_, name


def test_host_tensors_are_refused():
    import torch
    from dlprimitives_b200 import capi
    x, w, y = torch.zeros(4, 64), torch.zeros(64), torch.zeros(4, 64)
    q, s = torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(1, 4)
    for call in (lambda: capi.rms_norm(x, w, y), lambda: capi.quantize(x, q, s), lambda: capi.scaled_inner_product(q, s, q, s[:, :1], y),
                 lambda: capi.sample(x, w[:4], torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_binding_refuses_what_does_not_fit():
    """Shapes, types, strides and devices that do not fit each other."""
    import torch
    from dlprimitives_b200 import capi
    dev = "cuda:0"
    x, w, y = torch.zeros(4, 64, device=dev), torch.zeros(64, device=dev), torch.zeros(4, 64, device=dev)
    q, s, s1 = torch.zeros(4, 64, dtype=torch.float8_e4m3fn, device=dev), torch.zeros(1, 4, device=dev), torch.zeros(1, 1, device=dev)
    tokens, u, y4 = torch.zeros(4, dtype=torch.int32, device=dev), torch.zeros(4, device=dev), torch.zeros(4, 4, device=dev)
    capi.rms_norm(x, w, y)
    capi.rms_norm(x, w, q, scales=s)
    capi.quantize(x, q, s)
    capi.scaled_inner_product(q, s, q, s1, y4)
    capi.sample(x, u, tokens)
    for call in (lambda: capi.rms_norm(x, w[:63], y), lambda: capi.rms_norm(x, w.half(), y), lambda: capi.rms_norm(x.t(), u, y.t()),
                 lambda: capi.rms_norm(x, w, y[:3]), lambda: capi.rms_norm(x.int(), w, y), lambda: capi.rms_norm(x.cpu(), w, y),
                 lambda: capi.rms_norm(x, w.cpu(), y), lambda: capi.rms_norm(x, w, y, residual=x.half()), lambda: capi.rms_norm(x, w, y, residual=x, total=y[:2]),
                 lambda: capi.rms_norm(x, w, q, scales=s[:, :3]), lambda: capi.quantize(x, q, s.double()), lambda: capi.quantize(x, y, s),
                 lambda: capi.quantize(x, q, s, gate="silu"), lambda: capi.scaled_inner_product(q, s, q[:, :32], s1, y4),
                 lambda: capi.scaled_inner_product(q, s, q, s, y4), lambda: capi.scaled_inner_product(x, s, q, s1, y4),
                 lambda: capi.scaled_inner_product(q, s, q, s1, y4, bias=u[:3]), lambda: capi.scaled_inner_product(q, s, q, s1, tokens.view(4, 1)),
                 lambda: capi.sample(x, u, tokens.long()), lambda: capi.sample(x, u[:3], tokens), lambda: capi.sample(x, u, tokens, top_k=u),
                 lambda: capi.sample(x, x[:, 0], tokens)):
        with pytest.raises(ValueError):
            call()

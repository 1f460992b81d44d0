"""What the operators with typed operands refuse, before anything reaches a device: calls of the C ABI with made-up addresses."""
import pytest

A = 1 << 20                                          # an address with every alignment


def status(name, *args):
    from dlprimitives_b200 import capi
    return getattr(capi.lib(), name)(*args), capi.lib().dlp_last_error().decode()


def refused(name, good, changes):
    from dlprimitives_b200 import capi
    for change in changes:
        args = dict(good)
        args.update(change)
        st, msg = status(name, *args.values())
        assert st == capi.INVALID_ARGUMENT, change
        assert msg.startswith("Failed "), msg


def test_rms_norm():
    good = dict(x=A, xs=64, r=A, rs=64, total=A, ts=64, w=A, type=2, y=A, ys=64, y_type=3, scales=A, ss=8, rows=8, cols=64, eps=1e-5, stream=None)
    refused("dlp_rms_norm_fwd", good, [
        dict(x=None), dict(w=None), dict(y=None), dict(scales=None), dict(y_type=2), dict(r=None), dict(type=3), dict(type=-1), dict(y_type=4),
        dict(rows=-1), dict(cols=0), dict(xs=63), dict(rs=63), dict(ts=0), dict(ys=-64), dict(cols=200, xs=200, rs=200, ts=200, ys=200, ss=7),
        dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=A + 1), dict(w=A + 1), dict(total=A + 1), dict(scales=A + 2),
        dict(type=0, x=A + 2)])


def test_quantize():
    good = dict(x=A, xs=600, type=2, gate=1, q=A, qs=300, scales=A, ss=8, block_rows=1, rows=8, cols=300, stream=None)
    refused("dlp_quantize_fwd", good, [
        dict(x=None), dict(q=None), dict(scales=None), dict(type=3), dict(gate=3), dict(gate=-1), dict(block_rows=2), dict(block_rows=128),
        dict(xs=599), dict(qs=299), dict(ss=7), dict(rows=-1), dict(cols=0), dict(x=A + 1), dict(scales=A + 1),
        dict(gate=0, block_rows=128, rows=129, ss=2)])


def test_scaled_ip():
    good = dict(x=A, xs=304, x_scales=A, xss=8, w=A, ws=304, w_scales=A, wss=3, bias=None, y=A, ys=200, y_type=2, act=0, rows=8, inputs=300, outputs=200,
                stream=None)
    refused("dlp_scaled_ip_fwd", good, [
        dict(x=None), dict(x_scales=None), dict(w=None), dict(w_scales=None), dict(y=None), dict(xs=288), dict(xs=301), dict(ws=303), dict(ws=288),
        dict(x=A + 8), dict(w=A + 4), dict(xss=7), dict(wss=2), dict(ys=199), dict(y_type=3), dict(y_type=-1), dict(act=5), dict(act=-1), dict(rows=-1),
        dict(inputs=0), dict(outputs=0), dict(bias=A + 2), dict(y=A + 1), dict(x_scales=A + 2), dict(xs=1 << 41), dict(ws=1 << 41)])


def test_sample():
    good = dict(x=A, stride=100, type=0, rows=4, classes=100, t=None, k=None, p=None, m=None, u=A, tokens=A, stream=None)
    refused("dlp_sample_fwd", good, [
        dict(x=None), dict(u=None), dict(tokens=None), dict(stride=99), dict(type=3), dict(rows=-1), dict(classes=0), dict(classes=(1 << 22) + 1, stride=1 << 23),
        dict(x=A + 2), dict(u=A + 1), dict(k=A + 2), dict(tokens=A + 3), dict(t=A + 1)])


def test_nothing_to_do_needs_no_tensors():
    assert status("dlp_rms_norm_fwd", None, 8, None, 0, None, 0, None, 0, None, 8, 0, None, 0, 0, 8, 1e-5, None)[0] == 0
    assert status("dlp_quantize_fwd", None, 8, 0, 0, None, 8, None, 0, 1, 0, 8, None)[0] == 0
    assert status("dlp_scaled_ip_fwd", None, 16, None, 0, None, 16, None, 1, None, None, 8, 0, 0, 0, 16, 8, None)[0] == 0
    assert status("dlp_sample_fwd", None, 8, 0, 0, 8, None, None, None, None, None, None, None)[0] == 0


def test_binding_refuses_before_the_library():
    """Shapes, types and devices that do not fit each other; host tensors."""
    import torch
    from dlprimitives_b200 import capi
    if torch.cuda.is_available():
        dev = "cuda:0"
    else:
        pytest.MonkeyPatch().setattr(capi, "_device", lambda: 0)
        dev = "cpu"
    x, w, y = torch.zeros(4, 64, device=dev), torch.zeros(64, device=dev), torch.zeros(4, 64, device=dev)
    q, s = torch.zeros(4, 64, dtype=torch.float8_e4m3fn, device=dev), torch.zeros(1, 4, device=dev)
    tokens, u = torch.zeros(4, dtype=torch.int32, device=dev), torch.zeros(4, device=dev)
    for call in (lambda: capi.rms_norm(x, w[:63], y), lambda: capi.rms_norm(x, w.half(), y), lambda: capi.rms_norm(x.t(), w[:4], y.t()),
                 lambda: capi.rms_norm(x, w, y[:3]), lambda: capi.rms_norm(x.int(), w, y), lambda: capi.rms_norm(x.cpu(), w, y),
                 lambda: capi.rms_norm(x, w, q, scales=s[:, :3]), lambda: capi.quantize(x, q, s.double()), lambda: capi.quantize(x, y, s),
                 lambda: capi.quantize(x, q, s, gate="silu"), lambda: capi.scaled_inner_product(q, s, q[:, :32], s, y),
                 lambda: capi.scaled_inner_product(q, s, q, s[:, :2], y), lambda: capi.scaled_inner_product(x, s, q, s, y),
                 lambda: capi.sample(x, u, tokens.long()), lambda: capi.sample(x, u[:3], tokens), lambda: capi.sample(x, u, tokens, top_k=u)):
        with pytest.raises(ValueError):
            call()

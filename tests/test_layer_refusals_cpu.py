"""What the layer operators refuse, on the host: Python checks on CPU tensors and the C entry points' validation.

No kernel is launched: every call is refused (or only sizes a workspace) before the device is touched.
"""

import ctypes

import pytest
import torch

import oops_amd
from nested_standin import NestedTensor
from oops_amd import OOpsUnsupportedError, _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_cpu_tensors_are_unsupported():
    x, w = torch.randn(3, 8), torch.ones(8)
    i8, s = torch.zeros(3, 8, dtype=torch.int8), torch.ones(3)
    q, ld, st = torch.randn(2, 5, 8), torch.zeros(2), torch.zeros(2, 8, 8)
    for call in (lambda: oops_amd.rms_norm(x, 8, w), lambda: oops_amd.rms_norm_int8(x, 8, w),
                 lambda: oops_amd.quantize_int8(x), lambda: oops_amd.int8_linear(i8, s, i8, s),
                 lambda: oops_amd.linear_attention(q, q, q, ld),
                 lambda: oops_amd.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], ld, st)):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError):
            call()


def test_norm_shapes():
    x = torch.randn(3, 8)
    with pytest.raises(ValueError, match="residual"):
        oops_amd.rms_norm(x, 8, residual=torch.randn(1, 8))
    with pytest.raises(OOpsUnsupportedError, match="final dimension"):
        oops_amd.rms_norm(x, (3, 8))


def test_int8_linear_shapes():
    x, w = torch.zeros(2, 3, 8, dtype=torch.int8), torch.zeros(5, 8, dtype=torch.int8)
    xs, ws = torch.ones(2, 3), torch.ones(5)
    for bad, what in (((x, xs, w[:, :7], ws), "takes input"), ((x, xs[0], w, ws), "scale"), ((x, xs, w, ws[:4]), "scale"),
                      ((x, xs, w[0], ws), "takes input"), ((x, xs, w, ws, torch.ones(1)), "bias")):  # fmt: skip
        with pytest.raises(ValueError, match=what):
            oops_amd.int8_linear(*bad)


def test_linear_attention_shapes():
    q, v, ld = torch.randn(2, 3, 5, 8), torch.randn(2, 3, 5, 4), torch.zeros(3)
    st = torch.zeros(2, 3, 8, 4)
    for bad, what in (((q, q[:, :1], v, ld), "same leading shape"), ((q, q, v[:, :, :4], ld), "same leading shape"),
                      ((q, q, v, ld[:1]), "log_decay"), ((q, q, v, ld, st[:1]), "state"),
                      ((q[0, 0], q[0, 0], v[0, 0], ld), "same leading shape"),
                      ((q, q, v, ld, None, torch.zeros(3, dtype=torch.int32)), "lengths")):  # fmt: skip
        with pytest.raises((ValueError, OOpsUnsupportedError), match=what if len(bad) < 6 else None):
            oops_amd.linear_attention(*bad)
    with pytest.raises(ValueError, match="state"):
        oops_amd.linear_attention_step(q[:, :, 0], q[:, :, 0], v[:, :, 0], ld, st[0])


FAKE = ctypes.c_void_p(256)


def _refused(lib, rc, code, what):
    assert rc == code, rc
    assert what in lib.oops_last_error().decode(), lib.oops_last_error()


def test_rms_norm_entry_points(lib):
    def geo(**kw):
        g = _lib.RmsNormGeometry(_lib.BF16, 1, 64, 1e-6, 4, 64, 64)
        for name, value in kw.items():
            setattr(g, name, value)
        return ctypes.byref(g)

    forward = lambda g, x=FAKE, r=None, s=None: lib.oops_rms_norm_forward(g, x, r, None, FAKE, s, None, None)  # noqa: E731
    for kw, what in (({"dtype": 9}, "dtype"), ({"width": 0}, "width"), ({"width": 16385}, "width"), ({"rows": -1}, "rows"),
                     ({"x_row": 63}, "strides")):  # fmt: skip
        _refused(lib, forward(geo(**kw)), 1, what)
    _refused(lib, forward(geo(), x=None), 1, "non-NULL")
    _refused(lib, forward(geo(), r=FAKE), 1, "sum")
    _refused(lib, forward(geo(r_row=8), r=FAKE, s=FAKE), 1, "strides")
    _refused(lib, lib.oops_rms_norm_forward(None, FAKE, None, None, FAKE, None, None, None), 1, "NULL")
    assert forward(geo(rows=0), x=None) == 0  # nothing to do
    need = lib.oops_rms_norm_backward_workspace_bytes(geo(rows=100000))
    assert need > 0 and need % 256 == 0 and lib.oops_rms_norm_backward_workspace_bytes(geo(width=0)) == 0
    back = lambda g, ws, n: lib.oops_rms_norm_backward(g, FAKE, FAKE, None, FAKE, None, FAKE, FAKE, ws, n, None)  # noqa: E731
    _refused(lib, back(geo(rows=100000), FAKE, need - 1), 3, "workspace")
    _refused(lib, back(geo(rows=100000), ctypes.c_void_p(8), need), 3, "aligned")
    _refused(lib, back(geo(rows=0), FAKE, need), 1, "rows")
    _refused(lib, lib.oops_rms_norm_int8(geo(), FAKE, None, None, None, FAKE, None, None), 1, "non-NULL")
    _refused(lib, lib.oops_quantize_int8(geo(), FAKE, FAKE, None, None), 1, "non-NULL")


def test_int8_entry_point(lib):
    def geo(**kw):
        g = _lib.Int8Geometry(4, 8, 16, 16, 16, _lib.BF16, _lib.F32)
        for name, value in kw.items():
            setattr(g, name, value)
        return ctypes.byref(g)

    call = lambda g, x=FAKE: lib.oops_int8_linear(g, x, FAKE, FAKE, FAKE, None, FAKE, None, 0, None)  # noqa: E731
    for kw, what in (({"out_dtype": 5}, "dtype"), ({"bias_dtype": _lib.F16}, "bias"), ({"k": 131072}, "k must"),
                     ({"rows": -1}, "rows"), ({"n": 2**31}, "n ("), ({"x_row": 15}, "strides"),
                     ({"w_row": 8}, "strides")):  # fmt: skip
        _refused(lib, call(geo(**kw)), 1, what)
    _refused(lib, call(geo(), x=None), 1, "non-NULL")
    assert call(geo(rows=0)) == 0 and call(geo(n=0)) == 0


def test_linear_attention_entry_points(lib):
    def geo(**kw):
        g = _lib.LinearAttnGeometry(_lib.BF16, 2, 16, 16, 1, 8)
        g.scale = 1.0
        for name, value in kw.items():
            setattr(g, name, value)
        return g

    def forward(g, ld=FAKE):
        return lib.oops_linear_attn_forward(ctypes.byref(g), FAKE, FAKE, FAKE, ld, None, None, FAKE, None, None, 0, None)

    for kw, what in (({"dtype": 3}, "dtype"), ({"heads": 0}, "heads"), ({"key_size": 129}, "key_size"),
                     ({"value_size": 0}, "value_size"), ({"length": -1}, "length"), ({"batch": 2**30}, "too many")):  # fmt: skip
        _refused(lib, forward(geo(**kw)), 1, what)
    bad = geo()
    bad.stride[_lib.LA_K][2] = -1
    _refused(lib, forward(bad), 1, "negative stride")
    _refused(lib, forward(geo(), ld=None), 1, "non-NULL")
    assert forward(geo(batch=0)) == 0
    g = ctypes.byref(geo())
    _refused(lib, lib.oops_linear_attn_backward(g, FAKE, FAKE, FAKE, FAKE, None, None, None, None, None, FAKE, None, None,
                                                None, None, 0, None), 1, "grad_out")  # fmt: skip
    _refused(lib, lib.oops_linear_attn_step(g, FAKE, FAKE, FAKE, FAKE, None, FAKE, None), 1, "non-NULL")


def test_nested_operands():
    a = NestedTensor([torch.randn(n, 8) for n in (3, 5)], ragged_dims=(0,))
    i8, s = torch.zeros(5, 8, dtype=torch.int8), torch.ones(5)
    for call in (lambda: oops_amd.rms_norm_int8(a, 8), lambda: oops_amd.rms_norm_int8(a, 8, residual=a),
                 lambda: oops_amd.quantize_int8(a), lambda: oops_amd.int8_linear(a, s, i8, s),
                 lambda: oops_amd.linear_attention(a, a, a, s), lambda: oops_amd.linear_attention_step(a, a, a, s, s)):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError, match="dense"):
            call()
    for norm in (oops_amd.rms_norm, oops_amd.rms_norm_int8):
        with pytest.raises(ValueError, match="residual"):
            norm(a.concat, 8, residual=a)

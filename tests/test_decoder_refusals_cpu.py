"""What the decoder's operators refuse, on the host: Python checks on CPU tensors and the C entry points' validation.

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


def _cache(pages=2, heads=2, size=32, page=16):
    return oops_amd.quantized_cache(pages, heads, size, page_size=page, device="cpu")


def test_cpu_tensors_are_unsupported():
    q, k = torch.randn(4, 5, 32), torch.randn(2, 5, 32)
    table = oops_amd.rotary_table(5, 32, device="cpu")
    codes, scales = _cache()
    slots = torch.arange(5)
    for call in (lambda: oops_amd.causal_attention(q, k, k), lambda: oops_amd.rms_norm_rotary(q, k, table),
                 lambda: oops_amd.cache_write(codes, scales, k, k, slots), lambda: oops_amd.cache_read(codes, scales, slots),
                 lambda: oops_amd.cache_attention(q[:, 0], codes, scales, torch.zeros(2, dtype=torch.int32), torch.tensor(5))):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError):
            call()


def test_table_and_cache_on_the_host():
    t = oops_amd.rotary_table(3, 4, 100.0, device="cpu")
    a = torch.arange(3.0)[:, None] * torch.tensor([1.0, 0.1])
    torch.testing.assert_close(t, torch.stack((a.cos(), a.sin()), 1), rtol=0, atol=2.0**-23)
    codes, scales = _cache(3, 2, 96, 48)
    assert codes.shape == (3, 2, 2, 48, 48) and scales.shape == (3, 2, 2, 48, 3)
    assert codes.dtype == scales.dtype == torch.uint8 and not codes.any() and not scales.any()
    for bad in ((2, 2, 48, 16), (2, 2, 160, 16), (2, 2, 64, 24), (2, 2, 64, 0), (2, 2, 64, 1 << 21)):
        with pytest.raises(OOpsUnsupportedError):
            _cache(*bad)
    with pytest.raises(ValueError):
        _cache(2, 0)


def test_causal_attention_shapes():
    q, k, v = torch.randn(2, 4, 5, 8), torch.randn(2, 2, 5, 8), torch.randn(2, 2, 5, 4)
    for bad in ((q, k[:1], v), (q, k[:, :, :4], v), (q, k, v[:, :, :4]), (q[:, :3], k, v), (q, k[0], v), (q[0, 0], k[0, 0], v[0, 0]),
                (q, k[..., :7], v), (q, k, v, torch.zeros(0, dtype=torch.int32)), (q, k, v, torch.zeros(1, 3, dtype=torch.int32))):  # fmt: skip
        with pytest.raises(ValueError):
            oops_amd.causal_attention(*bad)
    with pytest.raises(OOpsUnsupportedError, match="int32 or int64"):
        oops_amd.causal_attention(q, k, v, torch.zeros(2))


def test_rotary_shapes():
    q, k, t = torch.randn(2, 4, 5, 8), torch.randn(2, 2, 5, 8), oops_amd.rotary_table(5, 8, device="cpu")
    for bad in ((q, k[:1], t), (q, k[:, :, :4], t), (q, k[0], t), (q, k, t[0]), (q, k, t[:, :1]), (q, k, oops_amd.rotary_table(5, 10, device="cpu")),
                (q, k, t, torch.zeros(3, 5, dtype=torch.int64)), (q, k, t, torch.zeros(1, 2, 5, dtype=torch.int64)),
                (q, k, t[:0], torch.zeros(5, dtype=torch.int64))):  # fmt: skip
        with pytest.raises(ValueError):
            oops_amd.rms_norm_rotary(*bad)
    with pytest.raises(OOpsUnsupportedError, match="int32 or int64"):
        oops_amd.rms_norm_rotary(q, k, t, torch.zeros(5))


def test_cache_shapes():
    codes, scales = _cache()
    k, slots, q = torch.randn(2, 5, 32), torch.arange(5), torch.randn(3, 4, 32)
    pages, n = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    for call in (lambda: oops_amd.cache_write(codes, scales[..., :0], k, k, slots), lambda: oops_amd.cache_write(codes[0], scales[0], k, k, slots),
                 lambda: oops_amd.cache_read(codes, scales[:1], slots), lambda: oops_amd.cache_attention(q, codes, scales[:, :1], pages, n)):  # fmt: skip
        with pytest.raises(ValueError, match="takes codes"):
            call()


def test_nested_operands():
    a = NestedTensor([torch.randn(n, 8) for n in (3, 5)], ragged_dims=(0,))
    t, (codes, scales), s = oops_amd.rotary_table(5, 8, device="cpu"), _cache(), torch.arange(5)
    for call in (lambda: oops_amd.causal_attention(a, a, a), lambda: oops_amd.rms_norm_rotary(a, a, t),
                 lambda: oops_amd.cache_write(codes, scales, a, a, s), lambda: oops_amd.cache_attention(a, codes, scales, s, s)):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError, match="dense"):
            call()


FAKE = ctypes.c_void_p(256)


def _refused(lib, rc, code, what):
    assert rc == code, rc
    assert what in lib.oops_last_error().decode(), lib.oops_last_error()


def _set(g, kw):
    for name, value in kw.items():
        setattr(g, name, value)
    return g


def test_rotary_entry_points(lib):
    def geo(**kw):
        g = _lib.RotaryGeometry(_lib.BF16, 64, 64, 0)
        g.heads[:], g.batch, g.length, g.table_rows = (4, 2), 1, 8, 8
        return ctypes.byref(_set(g, kw))

    forward = lambda g, q=FAKE, t=FAKE: lib.oops_rms_norm_rotary_forward(g, q, FAKE, None, None, t, None, FAKE, FAKE, None)  # noqa: E731
    for kw, what in (({"dtype": 9}, "dtype"), ({"size": 0}, "size"), ({"size": 257}, "size"), ({"rotary": 66}, "rotary"), ({"rotary": 3}, "rotary"),
                     ({"heads": (ctypes.c_int32 * 2)(4, 0)}, "heads"), ({"length": -1}, "length"), ({"batch": 2**30}, "length"),
                     ({"table_rows": 0}, "table")):  # fmt: skip
        _refused(lib, forward(geo(**kw)), 1, what)
    _refused(lib, forward(geo(), q=None), 1, "non-NULL")
    _refused(lib, forward(geo(), t=None), 1, "non-NULL")
    _refused(lib, forward(None), 1, "NULL")
    assert forward(geo(batch=0), q=None) == 0
    need = lib.oops_rms_norm_rotary_backward_workspace_bytes(geo(length=100000, table_rows=100000))
    assert need > 0 and need % 256 == 0 and lib.oops_rms_norm_rotary_backward_workspace_bytes(geo(size=0)) == 0

    def back(g, ws, n, dy=FAKE):
        return lib.oops_rms_norm_rotary_backward(g, FAKE, FAKE, FAKE, FAKE, FAKE, None, dy, FAKE, FAKE, FAKE, FAKE, FAKE, ws, n, None)

    _refused(lib, back(geo(length=100000), FAKE, need - 1), 3, "workspace")
    _refused(lib, back(geo(length=100000), ctypes.c_void_p(8), need), 3, "aligned")
    _refused(lib, back(geo(), FAKE, need, None), 1, "gradient of the inputs")
    _refused(lib, back(geo(batch=0), FAKE, need), 1, "tokens")


def test_causal_entry_points(lib):
    def geo(**kw):
        g = _lib.CausalGeometry(_lib.BF16, 4, 2, 64, 64, 0, 0, 0.125, 1, 8)
        for i in range(_lib.CA_OPERANDS):
            g.stride[i][:] = (8 * 4 * 64, 64, 4 * 64)
        return _set(g, kw)

    def forward(g, q=FAKE, ws=None, n=0, offsets=None):
        return lib.oops_causal_attn_forward(ctypes.byref(g), q, FAKE, FAKE, offsets, FAKE, None, None, ws, n, None)

    for kw, what in (({"dtype": 3}, "dtype"), ({"heads": 3}, "heads"), ({"kv_heads": 0}, "heads"), ({"key_size": 136}, "key_size"),
                     ({"key_size": 12}, "key_size"), ({"value_size": 0}, "value_size"), ({"length": -1}, "batch"), ({"batch": 2**23}, "2^24"),
                     ({"length": 2**31}, "batch")):  # fmt: skip
        _refused(lib, forward(geo(**kw)), 1, what)
    for values, what in (((64, -1, 64), "negative"), ((64, 64, 1 << 23), "2^24 bytes"), ((64, 4, 64), "16-byte"), ((64, 64, 3), "16-byte")):
        bad = geo()
        bad.stride[_lib.CA_K][:] = values
        _refused(lib, forward(bad), 1, what)
    one = geo(kv_heads=1)  # (the stride of a single head is nobody's)
    one.stride[_lib.CA_K][:] = (64, 3, 64)
    _refused(lib, forward(one, q=None), 1, "non-NULL")
    _refused(lib, forward(geo(), q=None), 1, "non-NULL")
    _refused(lib, forward(geo(), q=ctypes.c_void_p(264)), 1, "16 bytes")
    _refused(lib, forward(geo(sequences=-1), offsets=FAKE), 1, "sequences")
    assert forward(geo(batch=0), q=None) == 0 and forward(geo(length=0), q=None) == 0
    # packed blocks that are more than the chip's places are put in order first
    many = geo(length=1 << 16, sequences=3)
    need = lib.oops_causal_attn_forward_workspace_bytes(ctypes.byref(many))
    assert need == (1 << 16) // 128 * 2 * 4 and lib.oops_causal_attn_forward_workspace_bytes(ctypes.byref(geo(sequences=3))) == 0
    _refused(lib, forward(many, offsets=FAKE), 3, "workspace")
    # few workgroups' walks are split: their parts of the output, and two statistics of each
    few = geo(length=1024)
    need = lib.oops_causal_attn_forward_workspace_bytes(ctypes.byref(few))
    assert need == 4 * (4 * 1024 * 64 * 4 + 4 * 1024 * 2 * 4)
    _refused(lib, forward(few), 3, "workspace")
    _refused(lib, forward(few, ws=FAKE, n=need - 1), 3, "workspace")
    need = lib.oops_causal_attn_backward_workspace_bytes(ctypes.byref(geo()))
    stats, parts = 2 * 256, 2 * 8 * 2 * 64 * 4 * 2  # lse and delta; two parts of dk and of dv
    assert need == stats + parts

    def back(g, ws, n, dout=FAKE):
        return lib.oops_causal_attn_backward(ctypes.byref(g), FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, dout, FAKE, FAKE, FAKE, ws, n, None)

    _refused(lib, back(geo(), FAKE, need - 1), 3, "workspace")
    _refused(lib, back(geo(), FAKE, need, None), 1, "grad_out")


def test_cache_entry_points(lib):
    def geo(**kw):
        return _set(_lib.CacheGeometry(_lib.BF16, 2, 64, 16, 1, 4, 1, 8), kw)

    def write(g, key=FAKE, codes=FAKE, ws=None, n=0):
        return lib.oops_cache_write(ctypes.byref(g), codes, FAKE, key, FAKE, FAKE, ws, n, None)

    for kw, what in (({"dtype": 3}, "dtype"), ({"heads": 0}, "heads"), ({"heads": 1 << 17}, "heads"), ({"size": 48}, "size"), ({"size": 160}, "size"),
                     ({"page": 24}, "page"), ({"page": 0}, "page"), ({"pages": 2**28}, "pages"), ({"length": -1}, "length"),
                     ({"length": 2**28}, "too many")):  # fmt: skip
        _refused(lib, write(geo(**kw)), 1, what)
    _refused(lib, write(geo(), key=None), 1, "non-NULL")
    _refused(lib, write(geo(), codes=ctypes.c_void_p(260)), 1, "16 bytes")
    assert write(geo(length=0), key=None) == 0 and write(geo(pages=0), key=None) == 0
    assert lib.oops_cache_write_workspace_bytes(ctypes.byref(geo())) == 0
    need = lib.oops_cache_write_workspace_bytes(ctypes.byref(geo(length=5000)))
    assert need == 4 * 16 * 4
    _refused(lib, write(geo(length=5000)), 3, "workspace")
    odd = geo()
    odd.stride[0][:] = (0, 64, 132)
    _refused(lib, lib.oops_cache_read(ctypes.byref(odd), FAKE, FAKE, FAKE, FAKE, FAKE, None), 1, "strides")

    def attend(table=FAKE, ws=None, n=0, **kw):
        g = _set(_lib.CacheAttnGeometry(_lib.BF16, 4, 2, 64, 16, 0, 4, 1, 4), kw)
        return lib.oops_cache_attn(ctypes.byref(g), FAKE, FAKE, FAKE, table, FAKE, FAKE, ws, n, None)

    for kw, what in (({"dtype": 3}, "dtype"), ({"heads": 3}, "heads"), ({"kv_heads": 0}, "heads"), ({"size": 40}, "size"), ({"page": 8}, "page"),
                     ({"max_pages": 2**28}, "max_pages"), ({"batch": 2**21}, "batch"), ({"batch": -1}, "batch")):  # fmt: skip
        _refused(lib, attend(**kw), 1, what)
    _refused(lib, attend(table=None), 1, "non-NULL")
    _refused(lib, attend(max_pages=1000), 3, "workspace")
    assert attend(batch=0) == 0

"""The head's float64 restatement on a worked example, and argument errors of include/et_logit_head.h that
need no device."""
import ctypes

import numpy as np

from oracle import head_oracle as HO
from test_capi_symbols import ROOT, declared


def test_header_and_bindings_agree():
    from executorch_amd import _capi

    names = declared(f"{ROOT}/include/et_logit_head.h")
    assert sorted(_capi.HEAD_SIGNATURES) == names
    lib = ctypes.CDLL(_capi.LIB_PATH)
    for name in names:
        assert hasattr(lib, name), name


def test_worked_example():
    # one row of five weights in two groups (of three columns, here): nibbles 8 9 7 15 0
    packed = np.array([[0x98, 0xF7, 0x00]], dtype=np.uint8)
    x = np.array([[1.0, 2.0, 4.0, 8.0, 16.0]])
    y, bound = HO.logits(x, packed, np.array([[0.5, 2.0]]), np.array([[0.25, -1.0]]), 3, "f32")
    # (0 + 2 - 4) * 0.5 + 7 * 0.25 + (56 - 128) * 2 - 24
    assert y[0, 0] == -1.0 + 1.75 - 144.0 - 24.0
    assert 0 < bound[0, 0] < 0.01


def test_create_refusals_need_no_device():
    from executorch_amd import _capi

    L = _capi.lib()
    h = ctypes.c_void_p()
    one = ctypes.c_void_p(1 << 20)  # (never read: every call here is refused before that)

    def create(vocab=64, hidden=128, group=32, packed=one, stride=64, scales=one, zeros=None, dtype=_capi.DTYPE_FLOAT):
        return L.ets_logit_head_create(vocab, hidden, group, packed, stride, scales, zeros, dtype, None, ctypes.byref(h))

    for kw, word in (({"vocab": 0}, b"vocab_size"), ({"hidden": 0}, b"hidden_size"), ({"group": 0}, b"group_size"), ({"group": 96}, b"group_size"),
                     ({"group": -128}, b"group_size"), ({"group": 16}, b"group_size"), ({"packed": None}, b"null"), ({"scales": None}, b"null"),
                     ({"stride": 63}, b"shorter"), ({"dtype": _capi.DTYPE_UINT16}, b"scale type"), ({"scales": ctypes.c_void_p(3)}, b"aligned"),
                     ({"zeros": ctypes.c_void_p(5)}, b"aligned")):
        assert create(**kw) == _capi.INVALID_ARGUMENT, kw
        assert word in L.ets_logit_head_last_error(None), kw
    assert create(vocab=1 << 24) == _capi.NOT_SUPPORTED and create(hidden=(1 << 20) + 1, stride=1 << 20) == _capi.NOT_SUPPORTED
    assert L.ets_logit_head_create(64, 128, 32, one, 64, one, None, 6, None, None) == _capi.INVALID_ARGUMENT
    assert L.ets_logit_head_logits(None, one, 6, 1, 128, one, 6, 64, None) == _capi.INVALID_ARGUMENT
    assert L.ets_sampler_sample_hidden(None, None, one, 6, 1, 128, one, 6, 64, one, None) == _capi.INVALID_ARGUMENT
    assert L.ets_logit_head_destroy(None) == _capi.OK

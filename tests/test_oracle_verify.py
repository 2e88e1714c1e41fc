"""The verification oracle against known answers and against the distribution it has to give; argument
errors of include/et_speculative.h that need no device."""
import ctypes

import numpy as np
import pytest

from oracle import verify_oracle as VO
from test_capi_symbols import ROOT, declared


def test_header_and_bindings_agree():
    from executorch_amd import _capi

    names = declared(f"{ROOT}/include/et_speculative.h")
    assert sorted(_capi.SPECULATIVE_SIGNATURES) == names
    lib = ctypes.CDLL(_capi.LIB_PATH)
    for name in names:
        assert hasattr(lib, name), name
    # the struct as a C compiler lays it out on this ABI: 8-byte pointers and strides, no padding between
    assert ctypes.sizeof(_capi.VerifyBatch) == 136
    assert _capi.VerifyBatch.target_sequence_stride.offset == 32


def test_create_refusals_need_no_device():
    from executorch_amd import _capi

    L = _capi.lib()
    h = ctypes.c_void_p()
    for args, code, word in (((0, 1, 1), _capi.INVALID_ARGUMENT, b"vocab_size"), ((10, 0, 1), _capi.INVALID_ARGUMENT, b"max_sequences"),
                             ((10, 1, -1), _capi.INVALID_ARGUMENT, b"max_drafts"), ((10, 1, 65), _capi.NOT_SUPPORTED, b"max_drafts"),
                             ((1 << 24, 1, 1), _capi.NOT_SUPPORTED, b"vocab_size"),
                             ((1 << 23, 65535, 64), _capi.NOT_SUPPORTED, b"too large"),
                             ((2048 * 257, 65535, 0), _capi.NOT_SUPPORTED, b"too large")):
        assert L.ets_verifier_create(*args, ctypes.byref(h)) == code, args
        assert word in L.ets_verifier_last_error(None), args
    assert L.ets_verifier_create(10, 1, 1, None) == _capi.INVALID_ARGUMENT
    assert L.ets_verifier_verify(None, None, None) == _capi.INVALID_ARGUMENT
    assert L.ets_verifier_destroy(None) == _capi.OK


def test_known_answers():
    V = 8
    flat = np.zeros((2, V))
    # p uniform, a looked-up draft: accepted exactly for coins below 1/8, and the draw is floor(8 c)
    for coin, kept in ((0.0, 1), (0.1249, 1), (0.125, 0), (0.9, 0)):
        tokens, n = VO.verify_one(flat, None, [3], 1, 1.0, [coin, 0.5], 1)
        assert n == kept
        assert tokens.tolist() == ([3, 4] if kept else [4, -1])  # without token 3: the mass 3.5 of 7 lies in entry 4
    assert VO.draw(np.array([0.0, 1.0, 0.0, 1.0]), 0.0) == 1
    assert VO.draw(np.array([0.0, 1.0, 0.0, 1.0]), 1.0) == 3
    assert VO.argmax(np.array([np.nan, -np.inf, 2.0, 2.0])) == 2 and VO.argmax(np.full(3, np.nan)) == 0


@pytest.mark.parametrize("with_draft", [True, False])
def test_tokens_are_distributed_as_the_target(with_draft):
    """One draft from q, verified: the first token of the answer is distributed as p whatever q is."""
    rng = np.random.default_rng(5)
    V, N = 6, 40000
    target, draft = rng.standard_normal((2, V)) * 1.5, rng.standard_normal((1, V)) * 1.5
    p, q = VO.probabilities(target[0], 0.8), VO.probabilities(draft[0], 0.8)
    counts = np.zeros(V)
    for x, u, w in zip(rng.choice(V, size=N, p=q), rng.random(N), rng.random(N)):
        tokens, n = VO.verify_one(target, draft if with_draft else None, [x], 1, 0.8, [u, w], 1)
        counts[tokens[0]] += 1
    # a binomial count deviates by 5 standard deviations with probability 6e-7
    assert (np.abs(counts - N * p) < 5 * np.sqrt(N * p * (1 - p))).all()

"""The 8-bit integer entry points refuse bad arguments before any HIP call (no
GPU here), and the binding refuses tensors that do not fit."""
import ctypes

import numpy as np
import pytest

import moe_ffn

F32, BF16 = moe_ffn.F32, moe_ffn.BF16


@pytest.fixture()
def buf():
    return (ctypes.c_float * 256)()


def test_quantise_arguments(buf):
    q = moe_ffn.library().moe_quantize_i8
    good = [buf, F32, 64, 64, 1, buf, buf, buf, None]
    for at, bad in ((0, None), (1, 3), (1, -1), (2, 63), (3, 0), (3, 16385), (4, 0), (4, 65537), (5, None), (6, None), (7, None)):
        args = list(good)
        args[at] = bad
        assert q(*args) == 1, (at, bad)
    odd = ctypes.c_void_p(ctypes.addressof(buf) + 2)
    assert q(odd, F32, 64, 64, 1, buf, buf, buf, None) == 1      # 4-byte elements on 2 bytes
    assert q(buf, F32, 64, 64, 1, buf, odd, buf, None) == 1
    assert q(buf, F32, 64, 64, 1, buf, buf, odd, None) == 1
    assert q(ctypes.c_void_p(ctypes.addressof(buf) + 1), BF16, 64, 64, 1, buf, buf, buf, None) == 1


def test_linear_arguments(buf):
    lib = moe_ffn.library()
    h = ctypes.c_void_p(1)
    for args in ((48, 8, 0), (0, 8, 0), (16416, 8, 0), (64, 0, 0), (64, 262145, 0), (64, 8, -1), (64, 8, 65537)):
        assert lib.moe_i8_linear_create(*args, buf, buf, 0, 0, ctypes.byref(h)) == 1, args
        assert h.value is None   # nothing is left to destroy
    assert lib.moe_i8_linear_create(64, 8, 0, None, buf, 0, 0, ctypes.byref(h)) == 1
    assert lib.moe_i8_linear_create(64, 8, 0, buf, None, 0, 0, ctypes.byref(h)) == 1
    assert lib.moe_i8_linear_create(64, 8, 0, buf, buf, 0, -1, ctypes.byref(h)) == 1
    assert lib.moe_i8_linear_create(64, 8, 0, buf, buf, 0, 0, None) == 1
    assert lib.moe_i8_linear_forward(None, buf, buf, 1, buf, F32, 8, None) == 1
    assert lib.moe_i8_linear_apply(None, buf, F32, 64, 1, buf, F32, 8, buf, None) == 1
    assert lib.moe_i8_linear_destroy(None) == 1
    n = ctypes.c_size_t()
    assert lib.moe_i8_linear_bytes(None, ctypes.byref(n)) == 1


def test_bank_arguments(buf):
    lib = moe_ffn.library()
    h = ctypes.c_void_p(1)
    for args in ((0, 64, 8), (4097, 64, 8), (2, 48, 8), (2, 0, 8), (2, 16416, 8), (2, 64, 0), (2, 64, 65537)):
        assert lib.moe_i8_bank_create(*args, buf, buf, 0, 0, ctypes.byref(h)) == 1, args
        assert h.value is None
    assert lib.moe_i8_bank_create(2, 64, 8, None, buf, 0, 0, ctypes.byref(h)) == 1
    assert lib.moe_i8_bank_create(2, 64, 8, buf, None, 0, 0, ctypes.byref(h)) == 1
    assert lib.moe_i8_bank_create(2, 64, 8, buf, buf, 0, -1, ctypes.byref(h)) == 1
    assert lib.moe_i8_bank_create(2, 64, 8, buf, buf, 0, 0, None) == 1
    assert lib.moe_i8_bank_forward(None, buf, buf, 1, None, buf, 1, buf, F32, 8, buf, None) == 1
    assert lib.moe_i8_bank_destroy(None) == 1
    n = ctypes.c_size_t()
    assert lib.moe_i8_bank_bytes(None, ctypes.byref(n)) == 1


def test_layer_arguments(buf):
    lib = moe_ffn.library()
    good = dict(hidden=64, intermediate=32, experts=4, top_k=2, has_shared=1, max_tokens=8)
    bank = (moe_ffn.I8Matrix * 3)(*[moe_ffn.I8Matrix(ctypes.addressof(buf), ctypes.addressof(buf))] * 3)
    h, w, s = ctypes.c_void_p(1), ctypes.c_size_t(), ctypes.c_size_t()
    cfg = lambda **c: ctypes.byref(moe_ffn.I8LayerConfig(*{**good, **c}.values()))  # noqa: E731
    for bad in (dict(hidden=48), dict(hidden=0), dict(hidden=16416), dict(intermediate=16), dict(intermediate=16416),
                dict(experts=0), dict(experts=4096), dict(experts=4097, has_shared=0), dict(top_k=0), dict(top_k=5),
                dict(experts=64, top_k=33), dict(has_shared=2), dict(max_tokens=0), dict(max_tokens=65537)):
        assert lib.moe_i8_layer_create(cfg(**bad), bank, bank, 0, 0, ctypes.byref(h)) == 1, bad
        assert h.value is None
        assert lib.moe_i8_layer_memory_bytes(cfg(**bad), ctypes.byref(w), ctypes.byref(s)) == 1, bad
    assert lib.moe_i8_layer_create(None, bank, bank, 0, 0, ctypes.byref(h)) == 1
    assert lib.moe_i8_layer_create(cfg(), None, bank, 0, 0, ctypes.byref(h)) == 1
    assert lib.moe_i8_layer_create(cfg(), bank, None, 0, 0, ctypes.byref(h)) == 1
    hole = (moe_ffn.I8Matrix * 3)(bank[0], moe_ffn.I8Matrix(ctypes.addressof(buf), None), bank[2])
    assert lib.moe_i8_layer_create(cfg(), hole, bank, 0, 0, ctypes.byref(h)) == 1
    assert lib.moe_i8_layer_create(cfg(), bank, hole, 0, 0, ctypes.byref(h)) == 1
    assert lib.moe_i8_layer_create(cfg(), bank, bank, 0, -1, ctypes.byref(h)) == 1
    assert lib.moe_i8_layer_destroy(None) == 1
    assert lib.moe_i8_layer_forward(None, buf, F32, buf, buf, 1, None, buf, buf, None) == 1
    assert lib.moe_i8_layer_memory_bytes(cfg(hidden=2048, intermediate=512, experts=511, top_k=10), ctypes.byref(w),
                                         ctypes.byref(s)) == 0
    least = 512 * (3 * 2048 * 512 + (2 * 512 + 2048) * 4)
    assert least <= w.value < least + 4 * 256


def test_binding_checks_weights():
    c, s = np.zeros((130, 256), np.int8), np.ones(130, np.float32)
    for codes, scales in ((c[:129], s), (c, s[:1]), (c.T, s), (c, s[:, None])):
        with pytest.raises(ValueError):
            moe_ffn.MoeI8Linear(256, 130, codes, scales)
    for codes, scales in ((c.astype(np.uint8), s), (c, s.astype(np.float64))):
        with pytest.raises(TypeError):
            moe_ffn.MoeI8Linear(256, 130, codes, scales)
    for codes, scales in ((c, s), (c[None], s), (np.stack([c, c]), s[None])):
        with pytest.raises(ValueError):
            moe_ffn.MoeI8Bank(2, 256, 130, codes, scales)


def test_binding_checks_shared():
    """A shared expert's three matrices where the layer has one, none where not."""
    kinds = [(np.zeros((2, r, c), np.int8), np.ones((2, r), np.float32)) for r, c in ((32, 64), (32, 64), (64, 32))]
    shared = [(c[0], s[0]) for c, s in kinds]
    for has, given in ((False, shared), (True, None), (True, shared[:2])):
        with pytest.raises(ValueError):
            moe_ffn.MoeI8Layer(64, 32, 2, 1, has, 4, *kinds, shared=given)


def test_quantise_binding_refusals():
    torch = pytest.importorskip("torch")
    for bad in (torch.zeros(64), torch.zeros((2, 3, 4)), np.zeros((2, 64), np.float32)):
        with pytest.raises(ValueError):
            moe_ffn.quantize_i8(bad)

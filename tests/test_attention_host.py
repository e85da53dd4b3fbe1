"""Attention without a GPU: what the entry points refuse, and the tests' own arithmetic."""
import ctypes

import numpy as np
import pytest

from spcomm3d_amd import _capi as capi
from spcomm3d_amd import device
from tests import _attention as ref


def test_null_handles_are_invalid_arg():
    lib, h, p = capi.load(), ctypes.c_void_p(), ctypes.c_void_p()
    heads, seqs = ctypes.byref(capi.HeadsArg()), ctypes.byref(capi.CacheSeqsArg())
    bad = capi.ERR_INVALID_ARG
    assert lib.spc3d_band_create(None, 0, None, None, 0, 0, ctypes.byref(h)) == bad
    assert lib.spc3d_band_create(None, 0, None, None, 0, 0, None) == bad
    assert lib.spc3d_band_destroy(None) == bad
    assert lib.spc3d_attend(None, None, heads, heads, heads, 1.0, heads, None) == bad
    assert lib.spc3d_attend_grad(None, None, *[heads] * 3, 1.0, heads, None, *[heads] * 4) == bad
    assert lib.spc3d_cache_create(None, capi.BF16, 1, 16, 1, 64, ctypes.byref(h)) == bad
    assert lib.spc3d_cache_create(None, capi.BF16, 1, 16, 1, 64, None) == bad
    assert lib.spc3d_cache_wrap(None, capi.F8, 1, 16, 1, 64, None, None, None, None, ctypes.byref(h)) == bad
    assert lib.spc3d_cache_destroy(None) == bad
    assert lib.spc3d_cache_device_ptrs(None, ctypes.byref(p), None, None, None) == bad
    assert lib.spc3d_cache_append(None, None, seqs, heads, heads, None, None, None) == bad
    assert lib.spc3d_cache_attend(None, None, seqs, heads, 1.0, 0, 0, heads, None) == bad
    assert h.value is None and lib.spc3d_last_error()


def test_plans_and_vectors_keep_their_two_types():
    assert capi.load().spc3d_kernel_variant(capi.BF16, 64) is None
    for name in ("bf16", "e4m3", np.float16):
        with pytest.raises(TypeError):
            device.dtype_code(name)
    assert device.dtype_code("f8") == capi.F64  # numpy's name


def test_bfloat16_bits():
    x = np.array([0, 1, -1, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 3.4e38, np.inf, -np.inf, np.nan], np.float32)
    got = device.from_bf16(device.to_bf16(x))
    want = np.array([0, 1, -1, 1, 1 + 2.0 ** -6, np.inf, np.inf, -np.inf, np.nan], np.float32)
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(device.to_bf16(x), ref.to_bits(x, "bf16"))


def test_e4m3_codes():
    assert ref.F8[0x7E] == 448 and ref.F8[0x08] == 2.0 ** -6 and ref.F8[1] == 2.0 ** -9 and np.isnan(ref.F8[0xFF])
    exact = np.delete(ref.F8, [127, 255])
    assert np.array_equal(ref.F8[ref.f8_codes(exact)], exact)
    assert ref.F8[ref.f8_codes([17.0, 19.0, 460.0, 1e9, -1e9, 2.0 ** -11])].tolist() == [16, 20, 448, 448, -448, 0]


@pytest.mark.parametrize("most,e", [(0, -40), (448, 0), (449, 1), (448.0 * 2 ** -3, -3), (1, -8), (1e-30, -40), (1e30, 40)])
def test_scales(most, e):
    assert ref.scale_for(np.float32(most)) == 2.0 ** e


@pytest.mark.parametrize("window,sinks", [(0, 0), (4, 2)])
def test_the_oracles_gradients_against_differences(window, sinks):
    rng = np.random.default_rng(1)
    rows, cols, scale = [5, 7], [8, 7], 0.4
    x = {n: rng.normal(size=(sum(rows if n == "q" else cols), 2 if n == "q" else 1, 8)) for n in "qkv"}
    w = rng.normal(size=x["q"].shape)

    def out(y, **kw):
        return ref.band(y["q"], y["k"], y["v"], rows, cols, window, sinks, scale, "f32", **kw)

    got = out(x, d_o=w, o_in=out(x)["o"][0])
    for n in "qkv":
        step, h = rng.normal(size=x[n].shape), 1e-5
        loss = [float((out({**x, n: x[n] + s * h * step})["o"][0] * w).sum()) for s in (1, -1)]
        assert abs((loss[0] - loss[1]) / (2 * h) - float((got["d" + n][0] * step).sum())) < 1e-8

"""The 8-bit paged cache without a GPU: what its calls refuse, and that the
tests' 64-bit model of its codes is the format."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import _kv8 as kv8


def create(dsd, heads=2, dim=64, page=16, capacity=4, fmt=0, arrays=None):
    out = ctypes.c_void_p()
    status = dsd.load_library().dsd_kv8_create(heads, dim, page, capacity, fmt, arrays,
                                               ctypes.byref(out))
    return status, dsd.load_library().dsd_last_error().decode()


@pytest.mark.parametrize("bad,what", [
    (dict(heads=0), "num_kv_heads"), (dict(heads=4097), "num_kv_heads"),
    (dict(dim=0), "head_dim"), (dict(dim=24), "head_dim"), (dict(dim=272), "head_dim"),
    (dict(page=0), "page_size"), (dict(page=8), "page_size"), (dict(page=272), "page_size"),
    (dict(capacity=-1), "capacity_pages"), (dict(capacity=1 << 30), "31 bits"),
    (dict(fmt=2), "format"), (dict(fmt=-1), "format"),
])
def test_create_refuses(dsd, bad, what):
    status, message = create(dsd, **bad)
    assert status == 1 and what in message


def test_create_refuses_arrays(dsd):
    for name in ("keys", "values", "key_scales", "value_scales", "token_counts"):
        given = {n: 4096 for n in ("keys", "values", "key_scales", "value_scales", "token_counts")}
        given[name] = 0
        status, message = create(dsd, arrays=dsd.Kv8Arrays(**{n: p or None for n, p in given.items()}))
        assert status == 1 and "non-null" in message
        given[name] = 4104
        status, message = create(dsd, arrays=dsd.Kv8Arrays(**given))
        assert status == 1 and "16-byte" in message
    assert dsd.load_library().dsd_kv8_create(2, 64, 16, 4, 0, None, None) == 1


def test_null_handles_are_refused(dsd):
    lib = dsd.load_library()
    batch = dsd.Kv8Batch(1)
    assert lib.dsd_kv8_reset(None) == 1
    assert lib.dsd_kv8_destroy(None) == 0
    assert lib.dsd_kv8_device_arrays(None, None) == 1
    assert lib.dsd_kv8_set_rotation(None, 0, 0, None, 1.0) == 1
    assert lib.dsd_kv8_append(None, batch.pointer, 0, 0, None, 0, None, 0, None, 0, None, 0, None,
                              None) == 1
    assert lib.dsd_kv8_attend(None, batch.pointer, 0, 1, None, 0, None, 0, 0.0, None, 0, None,
                              None) == 1
    assert lib.dsd_kv8_attend_prompt(None, batch.pointer, 0, 1, None, 0, None, 0, 0.0, None, 0,
                                     None, None) == 1
    assert lib.dsd_kv8_workspace_bytes(None, batch.pointer, 1, None) == 1
    out = ctypes.c_void_p()
    assert lib.dsd_kv8_sparse_create(None, 1, 1, 1, 1, ctypes.byref(out)) == 1
    assert lib.dsd_kv8_sparse_create(None, 1, 1, 1, 1, None) == 1
    assert lib.dsd_kv8_sparse_destroy(None) == 0
    assert lib.dsd_kv8_sparse_status(None) == 1
    assert lib.dsd_kv8_sparse_run(None, 1, 1, 1, 0, None, 0, None, None, None, 0, None, None,
                                  None) == 1


def test_no_gpu_is_an_error(dsd):
    if dsd.gpu_available():
        pytest.skip("a GPU is visible")
    with pytest.raises(dsd.RuntimeFailure, match="gfx950"):
        dsd.Kv8Cache(2, 64, 16, 4)


def test_model_is_the_format():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(kv8.numbers(kv8.E4M3, codes.numpy()), want, equal_nan=True)
    # nearest() against torch's rounding, at random numbers, halves and subnormals
    rng = np.random.default_rng(5)
    x = np.concatenate([rng.standard_normal(4000) * 60, rng.standard_normal(4000) * 0.004,
                        (want[np.isfinite(want)][:-1] + want[np.isfinite(want)][1:]) / 2,
                        [0.0, -0.0, 448.0, 460.0, -500.0, 2.0 ** -10, 2.0 ** -11]])
    x = x.astype(np.float32).astype(np.float64)
    inside = np.clip(x, -448, 448)
    got = torch.from_numpy(inside).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(kv8.nearest(kv8.E4M3, x), got)
    assert np.isnan(kv8.nearest(kv8.E4M3, np.array([np.nan])))[0]
    assert kv8.nearest(kv8.INT8, np.array([np.nan, 0.5, 1.5, -2.5, 300.0])).tolist() == [0, 0, 2, -2, 127]


def test_model_scales():
    for fmt in (kv8.E4M3, kv8.INT8):
        most = np.array([0.0, 1e-45, 1e-30, 1.0, 3.5, 448.0, 448.1, 7e9, 3e38])
        scale = kv8.scale_for(fmt, most).astype(np.float64)
        assert (scale >= 2.0 ** -126).all()
        # the largest number's code is the largest one or, of e4m3, above half of it
        code = kv8.nearest(fmt, most.astype(np.float32) / scale)
        fits = most > 1e-30
        assert (code[fits] <= kv8.LARGEST[fmt]).all()
        assert (code[fits] > (220 if fmt == kv8.E4M3 else 126)).all()

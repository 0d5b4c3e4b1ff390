"""AdamW's refusals that need no GPU, and its 8-bit format's restatement."""
import ctypes as C

import numpy as np
import pytest
import torch

from tacotron2_amd import _lib
from tests import adamw_ref as ref


def test_library_refuses_bad_arguments_before_any_device_work():
    lib = _lib.load()
    ctx, out, buf = C.create_string_buffer(64), C.c_void_p(), C.create_string_buffer(64)
    at = (C.addressof(buf) + 15) & ~15
    sizes, decay = (C.c_int64 * 2)(5, 200), (C.c_double * 2)(0.0, 0.1)

    def create(**kw):
        a = dict(ctx=ctx, n=2, sizes=sizes, decay=decay, b1=0.9, b2=0.999, eps=1e-8, bits=32, seed=0, m=at, v=at, ms=None, vs=None, step=at, out=C.byref(out))
        a.update(kw)
        return lib.t2_adamw_create(*a.values())
    for kw in ({"ctx": None}, {"n": 0}, {"sizes": None}, {"decay": None}, {"b1": 1.0}, {"b1": -0.1}, {"b2": 1.0}, {"b2": float("nan")}, {"eps": 0.0}, {"bits": 16},
               {"bits": 8}, {"m": None}, {"v": None}, {"m": at + 4}, {"step": None}, {"out": None}, {"sizes": (C.c_int64 * 2)(5, 0)},
               {"sizes": (C.c_int64 * 2)(5, 1 << 41)}, {"decay": (C.c_double * 2)(0.0, -1.0)}, {"decay": (C.c_double * 2)(0.0, float("nan"))}):
        assert create(**kw) == _lib.T2_EINVAL, kw
    assert lib.t2_adamw_elements(2, sizes) == 128 + 256
    assert lib.t2_adamw_elements(1, (C.c_int64 * 1)(1 << 33)) == 1 << 33
    assert lib.t2_adamw_elements(1, (C.c_int64 * 1)((1 << 37) - 8192)) > 0 and lib.t2_adamw_elements(1, (C.c_int64 * 1)(1 << 37)) < 0    # a launch's threads
    assert lib.t2_adamw_step(None, None, None, 0.0, None, 0.0, 1.0, 0) == _lib.T2_EINVAL and lib.t2_adamw_step(ctx, None, None, 0.0, None, 0.0, 1.0, 0) == _lib.T2_EINVAL
    assert lib.t2_adamw_bind(ctx, None, None, None, None, None, None, None, None) == _lib.T2_EINVAL
    assert lib.t2_adamw_global_norm(ctx, None, None, 1.0, None) == _lib.T2_EINVAL and lib.t2_adamw_table_bytes(None) < 0
    assert lib.t2_adamw_destroy(None) == _lib.T2_OK


def test_codes_are_e4m3_and_rounding_is_unbiased():
    every = np.array([c for c in range(256) if c & 0x7F != 0x7F], np.uint8)
    assert np.array_equal(ref.e4m3(every), torch.from_numpy(every).view(torch.float8_e4m3fn).double().numpy())
    assert float(torch.tensor([120], dtype=torch.uint8).view(torch.float8_e8m0fnu).float()) == 2.0 ** (120 - 127)
    rng = np.random.default_rng(0)
    x = (rng.standard_normal(256) * np.exp2(rng.uniform(-12, 0, 256)) * 1e-3).astype(np.float32)
    x[5], x[200] = 0.0, 1e-12
    _, scale = ref.encode(x, np.zeros(256), False)
    power = np.repeat(2.0 ** (scale.astype(np.float64) - 127), 128)
    gap = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(x) / power, 1e-30))), -6.0) - 3.0) * power        # between neighbouring codes
    total = np.zeros(256)
    for w in range(0, 65536, 64):
        v = ref.decode(*ref.encode(x, np.full(256, w + 32), False))
        assert (np.abs(v - x) < gap).all()
        total += v
    # 1024 evenly spread words give the upper neighbour's probability in steps of a 1024th
    assert (np.abs(total / 1024 - x) <= gap / 1000).all()
    assert ref.decode(*ref.encode(x, np.zeros(256), False))[5] == 0.0
    # the largest value of a block never rounds beyond the format, exact values stay, a root above zero stays above it
    x = np.full(128, np.nextafter(np.float32(2), np.float32(1)))
    code, scale = ref.encode(x, np.full(128, 65535), True)
    assert ref.decode(code, scale).max() == 2.0 and code.max() < 0x7F
    x = np.full(128, 1e-30, np.float32)
    x[0] = 1.0
    assert (ref.decode(*ref.encode(x, np.zeros(128), True)) > 0).all()
    x = np.full(128, 1.0, np.float32)
    x[3] = np.nan
    code, scale = ref.encode(x, np.zeros(128), False)
    assert scale[0] == 255 and np.isnan(ref.decode(code, scale)).all()


def test_a_binding_serves_its_own_optimizer_only():
    """Its table has its optimizer's number of tensors: read by another's it would be left behind its end, or written past a tensor's."""
    from tacotron2_amd.training import AdamW, AdamWBinding

    def optimizer(sizes):
        o = AdamW.__new__(AdamW)
        o.sizes, o.spec, o.learning_rate, o.device, o._ctx, o._lib, o._h = sizes, None, 1e-3, torch.device("cuda", 0), None, None, C.c_void_p(16)
        return o
    few, many = optimizer([4]), optimizer([4, 4])
    b = AdamWBinding.__new__(AdamWBinding)
    b.table, b.grads, b.params, b.copies, b._raw, b._handle = torch.zeros(48, dtype=torch.uint8), [torch.zeros(4)], [torch.zeros(4)], None, 0, few._h
    same = optimizer([4])
    for other in (many, same):
        with pytest.raises(ValueError):
            other.apply_gradients(b)
        with pytest.raises(ValueError):
            other.global_norm(b)
    few._h = None                                            # closed
    with pytest.raises(ValueError):
        few.apply_gradients(b)
    for o in (few, many, same):
        o._h = None                                          # nothing of the library's to give back


def test_factors_that_are_no_numbers_are_refused():
    lib = _lib.load()
    nan, inf = float("nan"), float("inf")
    for lr, clip, scale, what in ((nan, 1.0, 1.0, b"learning_rate"), (inf, 1.0, 1.0, b"learning_rate"), (1e39, 1.0, 1.0, b"learning_rate"), (1e-3, nan, 1.0, b"clip_norm"),
                                  (1e-3, 1.0, nan, b"grad_scale"), (1e-3, 1.0, -inf, b"grad_scale"), (1e-3, 1.0, 1e39, b"grad_scale")):
        assert lib.t2_adamw_step(None, None, None, lr, None, clip, scale, 0) == _lib.T2_EINVAL and what in lib.t2_last_error(), what
    assert lib.t2_adamw_global_norm(None, None, None, nan, None) == _lib.T2_EINVAL and b"grad_scale" in lib.t2_last_error()


def test_an_epsilon_that_fp32_cannot_invert_is_refused():
    lib = _lib.load()
    ctx, out, buf = C.create_string_buffer(64), C.c_void_p(), C.create_string_buffer(64)
    at = (C.addressof(buf) + 15) & ~15
    for eps in (1e-46, 1e-39, 1.17e-38, 1e39, float("inf"), float("nan"), -1e-8):
        assert lib.t2_adamw_create(ctx, 1, (C.c_int64 * 1)(5), (C.c_double * 1)(0.0), 0.9, 0.999, eps, 32, 0, at, at, None, None, at, C.byref(out)) == _lib.T2_EINVAL, eps
        assert b"epsilon" in lib.t2_last_error()

"""The 8-bit format on the host against its definition in 64 bits, and the library's refusals that need no GPU."""
import ctypes

import numpy as np
import pytest
import torch

from nemo_amd import _lib, q8
from tests.q8_definition import decode, define, hard_rows


@pytest.mark.parametrize('c', [16, 112, 128, 144, 256, 400])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_host_follows_the_definition(c, dtype):
    x = hard_rows(257, c, seed=c).to(dtype)
    got = q8.quantize_host(x)
    codes, scale = define(x.double().numpy())
    assert np.array_equal(got.codes.double().numpy(), codes, equal_nan=True)
    assert np.array_equal(got.scale.double().numpy(), scale)
    back = q8.dequantize_host(got)
    with np.errstate(over='ignore'):   # the code above the largest f32 number stands for 2^128: infinity in f32
        assert np.array_equal(back.numpy(), decode(got.codes, got.scale).astype(np.float32), equal_nan=True)


def test_quantize_host_error_bound():
    x = torch.randn(500, 256, generator=torch.Generator().manual_seed(1))
    got = q8.quantize_host(x)
    back = q8.dequantize_host(got)
    # half a step of e4m3: 2^-4 of the number, or half of the smallest step, 2^-10 times the scale
    bound = torch.maximum(x.abs() * 2.0 ** -4, got.scale.float().repeat_interleave(128, -1) * 2.0 ** -10)
    assert bool(((back - x).abs() <= bound).all())


def test_quantize_host_keeps_what_is_representable():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    row = codes.float().nan_to_num(0.0)[None]          # all finite codes, amax 448 in either block: scale 1
    got = q8.quantize_host(row)
    assert torch.equal(got.scale.float(), torch.ones(1, 2)) and torch.equal(got.codes.float(), row)


def test_null_context_is_refused():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(64)
    assert lib.nemo_quantize(None, buf, 0, 0, 1, 1, 16, None, 1, buf, buf, None) == -1
    assert lib.nemo_dequantize(None, buf, buf, None, 1, 1, 1, 16, 0, 0, buf, None) == -1
    assert lib.nemo_q8_product(None, buf, buf, 1, buf, buf, 1, 16, 0, buf, None) == -1
    assert lib.nemo_q8_grouped_product(None, buf, buf, 1, buf, 1, buf, buf, 1, buf, 1, None, 16, 0, 1, buf, None) == -1
    assert lib.nemo_q8_clutter_score(None, buf, buf, 1, buf, buf, 1, None, 1, None, buf, None) == -1
    assert b'null ctx' in lib.nemo_last_error(None)

"""PoseEngine's 8-bit calls on the CPU: what they hand to the library, and what they refuse before it.  Tensors are on the meta device
(shapes without memory), the library is a list of calls."""
import numpy as np
import pytest
import torch

from nemo_amd import q8
from nemo_amd.engine import PoseEngine


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture
def eng():
    e = object.__new__(PoseEngine)
    e.device, e._gpu, e.ctx, e.lib, e.validate_indices = torch.device('meta'), -1, None, Recorder(), False
    e.h, e.w, e.D = 1, 1, 128
    e._raw_stream = lambda: 0
    return e


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device='meta')


def held(*shape):
    return q8.empty(shape, 'meta')


def index(n):
    return meta(n, dtype=torch.int32)


BIG = 2 ** 31
LOW = 2 ** 32 + 5   # its lower 32 bits are 5


@pytest.mark.parametrize('n', [BIG, LOW])
def test_sizes_that_an_int_does_not_hold_are_refused(eng, n):
    f16 = torch.float16
    for call in (lambda: eng.quantize(meta(n, 16, dtype=f16)),
                 lambda: eng.quantize(meta(2 ** 20, n // 2 ** 20 + 1, 16, dtype=f16)),
                 lambda: eng.quantize(meta(1, n, 16, dtype=f16), slots=index(1), out=held(3, n, 16)),
                 lambda: eng.quantize(meta(n, 16, 1, dtype=f16), channel_major=True),
                 lambda: eng.quantize(meta(1, 16, n, dtype=f16), channel_major=True),
                 lambda: eng.quantize(meta(1, n, dtype=f16)),
                 lambda: eng.quantize(meta(1, 16, dtype=f16), slots=index(1), out=held(n, 16)),
                 lambda: eng.dequantize(*held(n, 16)),
                 lambda: eng.dequantize(*held(1, n, 16), channel_major=True),
                 lambda: eng.dequantize(*held(n, 16), slots=index(1)),
                 lambda: eng.dequantize(*held(3, 16), slots=index(n)),
                 lambda: eng.dequantize(*held(1, n)),
                 lambda: eng.q8_product(held(1, 16), held(n, 16)),
                 lambda: eng.q8_product(held(1, n), held(1, n)),
                 lambda: eng.q8_grouped_product(held(1, 16), index(2), held(n, 16), index(2), n_cols=4),
                 lambda: eng.q8_grouped_product(held(1, 16), index(2), held(4, 16), index(2), n_cols=n),
                 lambda: eng.q8_grouped_product(held(1, 16), index(n + 1), held(4, 16), index(2)),
                 lambda: eng.q8_grouped_product(held(1, 16), index(2), held(4, 16), index(n + 1)),
                 lambda: eng.q8_grouped_product(held(1, n), index(2), held(4, n), index(2)),
                 lambda: eng.q8_clutter_score(held(n, 1, 1, 128), held(4, 128)),
                 lambda: eng.q8_clutter_score(held(1, 1, 1, 128), held(n, 128)),
                 lambda: eng.q8_clutter_score(held(1, 1, 1, 128), held(4, 128), index(n + 1), index(1))):
        with pytest.raises(ValueError, match='more than 2\\^31 - 1'):
            call()
    assert eng.lib.calls == []


def test_sizes_reach_the_library_whole(eng):
    eng.quantize(meta(3, 5, 7, 48))
    eng.quantize(meta(3, 48, 5, 7), channel_major=True)
    eng.quantize(meta(3, 5, 7, 48), slots=index(3), out=held(9, 5, 7, 48))
    eng.dequantize(*held(9, 5, 48))
    eng.dequantize(*held(9, 5, 48), channel_major=True)
    eng.dequantize(*held(9, 5, 48), slots=index(4))
    eng.q8_product(held(LOW, 16), held(3, 16))              # rows of a are 64 bits
    got = [(name[5:], a[3:7] + a[8:9] if name == 'nemo_quantize' else a[4:8] if name == 'nemo_dequantize' else (a[3],) + a[6:8]) for name, a in eng.lib.calls]
    assert got == [('quantize', (False, 1, 105, 48, 1)), ('quantize', (True, 3, 35, 48, 3)), ('quantize', (False, 3, 35, 48, 9)),
                   ('dequantize', (1, 1, 45, 48)), ('dequantize', (9, 9, 5, 48)), ('dequantize', (9, 4, 5, 48)), ('q8_product', (LOW, 3, 16))]


def test_what_is_no_tensor_is_refused(eng):
    q, b = held(1, 1, 1, 128), held(4, 128)
    for bad in ([1.0], np.zeros((4, 128), np.float32), 'out', 3):
        for call in (lambda: eng.quantize(bad), lambda: eng.quantize(meta(4, 128), out=bad), lambda: eng.quantize(meta(4, 128), out=(bad, bad)),
                     lambda: eng.quantize(meta(4, 128), slots=bad, out=b), lambda: eng.dequantize(bad, bad), lambda: eng.dequantize(*b, slots=bad),
                     lambda: eng.dequantize(*b, out=bad), lambda: eng.q8_product(bad, b), lambda: eng.q8_product(b, b, out=bad),
                     lambda: eng.q8_grouped_product(b, bad, b, index(2)), lambda: eng.q8_grouped_product(b, index(2), b, bad),
                     lambda: eng.q8_grouped_product(b, index(2), b, index(2), bank_of=bad), lambda: eng.q8_grouped_product(b, index(2), b, index(2), out=bad),
                     lambda: eng.q8_clutter_score(bad, b), lambda: eng.q8_clutter_score(q, b, bad), lambda: eng.q8_clutter_score(q, b, index(2), bad),
                     lambda: eng.q8_clutter_score(q, b, out=bad)):
            with pytest.raises(TypeError):
                call()
    assert eng.lib.calls == []

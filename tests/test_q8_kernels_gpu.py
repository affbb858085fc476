"""The 8-bit products and scores, each property on every kernel (tests/test_q8_plan_cpu.py holds that the sizes reach them).

Tolerances as in tests/test_q8_gpu.py: a product of K channels is off by at most K 2^-23 sum |a_c b_c|, a bf16 result by half a step more.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from nemo_amd import q8  # noqa: E402
from tests.q8_definition import decode  # noqa: E402
from tests.q8_reach import PRODUCTS, SCORES  # noqa: E402
from tests.test_q8_gpu import close, eng, offsets, rows8  # noqa: E402,F401


def coded(rows, k, seed, byte, top):
    """Rows of random codes below `top` with either sign, all scale bytes `byte`, and their numbers in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    c = (torch.randint(0, top, (rows, k), generator=g) | torch.randint(0, 2, (rows, k), generator=g) << 7).to(torch.uint8)
    q = q8.Q8(c.view(torch.float8_e4m3fn), torch.full((rows, q8.n_blocks(k)), byte, dtype=torch.uint8).view(torch.float8_e8m0fnu))
    return q8.Q8(q.codes.cuda(), q.scale.cuda()), torch.from_numpy(decode(*q))


@pytest.mark.parametrize('m,n,k', PRODUCTS)
def test_small_numbers(eng, m, n, k):  # noqa: F811
    """Subnormal codes down to the smallest scales: exact from 2^-133 on, multiples of it (ties to even) below."""
    for byte in (0, 2, 3, 9, 10):
        (a, a64), (b, b64) = coded(m, k, byte, byte, 16), coded(n, k, 50, 200, 127)
        close(eng.q8_product(a, b), torch.round(a64 * 2.0 ** 133) * 2.0 ** -133, b64, k)


@pytest.mark.parametrize('m,n,k', PRODUCTS)
def test_numbers_from_2_to_the_128_on_are_infinite(eng, m, n, k):  # noqa: F811
    (a, _), (b, _) = rows8(m, k, 1, spread=0), rows8(n, k, 2, spread=0)
    one = torch.zeros_like(a.codes.view(torch.uint8))
    one[:, k - 1] = 0x78                                                       # 256 with the scale below: 2^128
    a = q8.Q8(one.view(torch.float8_e4m3fn), torch.full_like(a.scale.view(torch.uint8), 247).view(torch.float8_e8m0fnu))
    b.codes.view(torch.uint8)[0, k - 1] = 0
    got, sign = eng.q8_product(a, b), torch.sign(eng.dequantize(*b)[:, k - 1])
    assert bool((got[:, sign > 0] == np.inf).all()) and bool((got[:, sign < 0] == -np.inf).all()) and bool(got[:, sign == 0].isnan().all())
    assert bool(got[:, 0].isnan().all()) and bool((eng.dequantize(*a)[:, k - 1] == np.inf).all())

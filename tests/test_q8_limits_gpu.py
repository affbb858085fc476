"""8-bit rows at the ends of the ranges that the calls accept."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from nemo_amd import _lib, q8  # noqa: E402
from tests.test_q8_gpu import close, eng, rows8  # noqa: E402,F401


@pytest.fixture(autouse=True)
def give_back():
    """Tests here hold up to a third of the memory."""
    yield
    torch.cuda.empty_cache()


def repeated(q, n):
    """n rows: those of q over and over."""
    out = q8.empty((n, q.codes.shape[1]), 'cuda')
    for to, part in zip(out, q):
        to, part = to.view(torch.uint8), part.view(torch.uint8)
        whole = n // len(part) * len(part)
        to[:whole].view(-1, *part.shape).copy_(part.expand(whole // len(part), *part.shape))
        to[whole:] = part[:n - whole]
    return out


def check_repeated(got, a64, b64, k):
    """Column j of the result is that of row j % len(b64): the first ones against 64 bits, the others equal to them."""
    p = len(b64)
    first = got[:, :p].contiguous()
    close(first, a64, b64, k)
    for m in range(got.shape[0]):
        whole = got.shape[1] // p * p
        assert bool((got[m, :whole].view(-1, p) == first[m]).all()), m
        assert torch.equal(got[m, whole:], first[m, :got.shape[1] - whole]), m


def test_widest_rows_of_a_result(eng):  # noqa: F811
    """64 rows of 2^27 numbers (34 GB): the rows of either half of a tile land where they belong; one column more is refused."""
    n = 1 << 27
    (a, a64), (b, b64) = rows8(64, 16, 1), rows8(4099, 16, 2)
    wide = repeated(b, n + 1)
    got = eng.q8_product(a, q8.Q8(wide.codes[:n], wide.scale[:n]))
    check_repeated(got, a64, b64, 16)
    del got
    out = torch.full((1, n + 1), 5.0, device='cuda')
    with pytest.raises(_lib.NemoHipError, match='at most 134217728'):
        eng.q8_product(q8.Q8(a.codes[:1], a.scale[:1]), wide, out=out)
    assert bool((out == 5.0).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('m,n,k', [(1, 65535 * 128 + 1, 16), (2, 65535 * 128 + 259, 128), (63, 65535 * 128 + 130, 32), (1, 65535 * 32 + 1, 272), (5, 65535 * 32 + 4000, 400)])
def test_few_rows_of_any_width(eng, m, n, k, dtype):  # noqa: F811
    (a, a64), (b, b64) = rows8(m, k, m + k), rows8(4099, k, k)
    check_repeated(eng.q8_product(a, repeated(b, n), dtype=dtype), a64, b64, k)


@pytest.mark.parametrize('m,n', [(2 ** 31 - 1023, 8), (2 ** 31 - 1, 8), (8, 2 ** 31 - 1)])
def test_more_rows_than_are_counted_are_refused(eng, m, n):  # noqa: F811
    (a, _), (b, _) = rows8(8, 128, 1), rows8(8, 128, 2)
    out = torch.full((8, 8), 5.0, device='cuda')
    off = torch.tensor([0, 8], dtype=torch.int32, device='cuda')
    at = [t.data_ptr() for t in (*a, *b, off, out)]
    assert eng.lib.nemo_q8_product(eng.ctx, at[0], at[1], m, at[2], at[3], n, 128, 0, at[5], None) < 0
    assert b'at most 2147482624' in eng.lib.nemo_last_error(eng.ctx)
    assert eng.lib.nemo_q8_grouped_product(eng.ctx, at[0], at[1], m, at[4], 1, at[2], at[3], n, at[4], 1, None, 128, 0, 8, at[5], None) < 0
    assert b'at most 2147482624' in eng.lib.nemo_last_error(eng.ctx)
    images = m // (eng.h * eng.w) + 1
    assert eng.lib.nemo_q8_clutter_score(eng.ctx, at[0], at[1], images, at[2], at[3], n, None, 1, None, at[5], None) < 0
    assert b'at most 2147482624' in eng.lib.nemo_last_error(eng.ctx)
    torch.cuda.synchronize()
    assert bool((out == 5.0).all())


def test_images_of_two_to_the_31_pixels_read_back(eng):  # noqa: F811
    """One image of 2^31 - 1 pixels, channels first: each channel ends at its own last pixel, and nothing is written behind the image."""
    rows, c = 2 ** 31 - 1, 16
    (part, part64) = rows8(4099, c, 3, spread=3)
    q = repeated(part, rows)
    flat = torch.full((rows * c + 64,), 123.0, dtype=torch.float16, device='cuda')
    got = eng.dequantize(q.codes[None], q.scale[None], channel_major=True, out=flat[:rows * c].view(1, c, rows))
    assert bool((flat[rows * c:] == 123.0).all())
    want, whole = part64.to(torch.float16).cuda(), rows // 4099 * 4099
    for k in range(c):
        assert bool((got[0, k, :whole].view(-1, 4099) == want[:, k]).all()), k
        assert torch.equal(got[0, k, whole:], want[:rows - whole, k]), k


@pytest.mark.parametrize('channel_major', [False, True])
def test_cache_without_slots(eng, channel_major):  # noqa: F811
    """Every slot is outside such a cache: nothing is written, zeros are read."""
    cache, slots = q8.empty((0, 5, 144), 'cuda'), torch.tensor([0, -1, 3], dtype=torch.int32, device='cuda')
    x = torch.randn((3, 144, 5) if channel_major else (3, 5, 144), device='cuda')
    assert eng.quantize(x, channel_major=channel_major, slots=slots, out=cache).codes.shape == (0, 5, 144)
    back = eng.dequantize(*cache, slots=slots, channel_major=channel_major, out=torch.full_like(x, 3.0))
    assert back.shape == x.shape and not bool(back.any())

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


@pytest.mark.parametrize('m,n,k', PRODUCTS)
def test_nan_stays_in_its_row_and_column(eng, m, n, k):  # noqa: F811
    """A NaN code in the last channel of the last row, of one in the middle and of the last column; byte 255 in the last block."""
    (a, a64), (b, b64) = rows8(m, k, 5), rows8(n, k, 6)
    rows, cols = [0, m // 2, m - 1], [n // 3, n - 1]
    a.codes.view(torch.uint8)[m - 1, k - 1] = 0x7f
    a.codes.view(torch.uint8)[m // 2, 0] = 0xff
    a.scale.view(torch.uint8)[0, -1] = 255
    b.codes.view(torch.uint8)[n - 1, k - 1] = 0xff
    b.scale.view(torch.uint8)[n // 3, -1] = 255
    for dtype in (torch.float32, torch.bfloat16):
        got = eng.q8_product(a, b, dtype=dtype)
        want = torch.zeros(m, n, dtype=torch.bool)
        want[rows], want[:, cols] = True, True
        assert torch.equal(got.isnan().cpu(), want)
        keep_m, keep_n = [torch.tensor([i for i in range(size) if i not in out]) for size, out in ((m, rows), (n, cols))]
        close(got[keep_m.cuda()][:, keep_n.cuda()], a64[keep_m], b64[keep_n], k)


@pytest.mark.parametrize('m,n,k', PRODUCTS)
def test_scales_of_any_size_meet_exactly(eng, m, n, k):  # noqa: F811
    """Scales of every row and block apart, up to 2^90 by 2^-90."""
    (a, _), (b, _) = rows8(m, k, 7, spread=0), rows8(n, k, 8, spread=0)
    g = torch.Generator().manual_seed(k)
    shift = lambda q, low: q8.Q8(q.codes, (q.scale.view(torch.uint8).int().cpu()  # noqa: E731
                                           + torch.randint(low, low + 20, q.scale.shape, generator=g)).to(torch.uint8).cuda().view(torch.float8_e8m0fnu))
    a, b = shift(a, -90), shift(b, 70)
    close(eng.q8_product(a, b), torch.from_numpy(decode(*a)), torch.from_numpy(decode(*b)), k)


@pytest.mark.parametrize('m,n,k', [s for s in PRODUCTS if s[2] <= 256])
def test_rows_do_not_depend_on_their_company(eng, m, n, k):  # noqa: F811
    """Up to 256 channels a row's products are the same bits on every kernel: alone, in groups, and in one large product."""
    (a, _), (b, _) = rows8(m, k, 21), rows8(n, k, 22)
    whole = eng.q8_product(a, b)
    for i in (0, m // 2 + 1, m - 1):
        assert torch.equal(whole[i:i + 1], eng.q8_product(q8.Q8(a.codes[i:i + 1].contiguous(), a.scale[i:i + 1].contiguous()), b)), i
    sizes = [3, 0, m // 3, 64]
    cut = eng.q8_grouped_product(a, offsets(sizes + [m - sum(sizes)]), b, offsets([n]), n_cols=n)
    assert torch.equal(whole, cut)
    narrow = eng.q8_product(a, q8.Q8(b.codes[:20].contiguous(), b.scale[:20].contiguous()))
    assert torch.equal(whole[:, :20], narrow[:, :n])


@pytest.mark.parametrize('m,n,k', PRODUCTS)
def test_captured_and_on_two_streams(eng, m, n, k):  # noqa: F811
    """Replays of a captured product, its bank and its rows changing between them, and two products at once, against eager calls, bit for bit."""
    data = [(rows8(m, k, s)[0], rows8(n, k, s + 9)[0]) for s in range(3)]
    want = [eng.q8_product(a, b) for a, b in data]
    hold = [q8.Q8(q.codes.clone(), q.scale.clone()) for q in data[0]]
    out, side, graph = torch.empty_like(want[0]), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eng.q8_product(*hold, out=out)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        eng.q8_product(*hold, out=out)
    for i in (1, 2, 0, 1):
        for to, new in zip(hold, data[i]):
            to.codes.view(torch.uint8).copy_(new.codes.view(torch.uint8))
            to.scale.view(torch.uint8).copy_(new.scale.view(torch.uint8))
        out.fill_(7.0)
        graph.replay()
        eager = eng.q8_product(*data[i])
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]) and torch.equal(eager, want[i])
    streams, got = [torch.cuda.Stream() for _ in range(2)], [torch.empty_like(w) for w in want[:2]]
    torch.cuda.synchronize()
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                eng.q8_product(*data[i], out=got[i])
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize('k,n', [(128, 300), (256, 300), (1024, 300)])
def test_rows_beyond_32_bits(eng, k, n):  # noqa: F811
    """The last rows of an operand of more than 4 GiB, on the short-row and the long-row kernel, and a result of more than 4 GiB."""
    rows = (1 << 32) // k + 9000
    a = q8.empty((rows, k), 'cuda')
    tail, tail64 = rows8(9000, k, 3)
    a.codes.view(torch.uint8)[:rows - 9000] = 0
    a.scale.view(torch.uint8)[:rows - 9000] = 127
    for to, part in zip(a, tail):
        to.view(torch.uint8)[rows - 9000:] = part.view(torch.uint8)
    b, b64 = rows8(n, k, 4)
    got = eng.q8_product(a, b)
    close(got[rows - 9000:], tail64, b64, k)
    assert not bool(got[:rows - 9000].any())
    del got
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------ scores
@pytest.fixture(params=SCORES, ids=str)
def maps(request):
    from nemo_amd.engine import PoseEngine
    n, h, w, d = request.param
    q, q64 = rows8(n * h * w, d, n + d)
    return PoseEngine(max(h, w, 24), (h, w), d), q8.Q8(q.codes.view(n, h, w, d), q.scale.view(n, h, w, d // 128)), q64, d


@pytest.mark.parametrize('rows', [1, 70, 300])
def test_score_keeps_nan(maps, rows):
    """NaN in one pixel stays there; NaN anywhere in the bank (its first and its last row, its first and its last channel) is everywhere."""
    eng, a, _, d = maps  # noqa: F811
    (b, _) = rows8(rows, d, 42)
    clean = eng.q8_clutter_score(a, b)
    assert not bool(clean.isnan().any())
    last = tuple(s - 1 for s in a.codes.shape[:3])
    for at in (last, (0, 0, 0), (last[0] // 2, last[1], 0)):
        kept = a.codes[at].view(torch.uint8).clone()
        a.codes.view(torch.uint8)[at][d - 1] = 0x7f
        got = eng.q8_clutter_score(a, b)
        assert bool(got[at].isnan()) and int(got.isnan().sum()) == 1
        got[at] = clean[at]
        assert torch.equal(got, clean)
        a.codes.view(torch.uint8)[at] = kept
    for r, c, byte in ((0, 0, None), (rows - 1, d - 1, None), (rows - 1, 0, 255)):
        bad = q8.Q8(b.codes.clone(), b.scale.clone())
        if byte is None:
            bad.codes.view(torch.uint8)[r, c] = 0xff
        else:
            bad.scale.view(torch.uint8)[r, -1] = byte
        assert bool(eng.q8_clutter_score(a, bad).isnan().all())


def test_score_of_each_map_alone_and_again(maps):
    """A map's scores are the same bits alone (the kernel for few pixels) and among others, captured or not."""
    eng, a, a64, d = maps  # noqa: F811
    (b, b64) = rows8(333, d, 43)
    n = a.codes.shape[0]
    got = eng.q8_clutter_score(a, b)
    want, bound = (a64 @ b64.t()).amax(1).view(got.shape), (d * 2.0 ** -23 * (a64.abs() @ b64.abs().t()).amax(1)).view(got.shape)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    for i in (0, n // 2, n - 1):
        assert torch.equal(got[i:i + 1], eng.q8_clutter_score(q8.Q8(a.codes[i:i + 1].contiguous(), a.scale[i:i + 1].contiguous()), b))
    out, side, graph = torch.empty_like(got), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eng.q8_clutter_score(a, b, out=out)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        eng.q8_clutter_score(a, b, out=out)
    for _ in range(3):
        out.fill_(7.0)
        graph.replay()
        again = eng.q8_clutter_score(a, b)
        torch.cuda.synchronize()
        assert torch.equal(out, got) and torch.equal(again, got)


# ------------------------------------------------------------------------------------------------ quantise and read back
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('n,pixels,c', [(3, 129, 128), (2, 255, 144), (3, 777, 48), (2, 1023, 256), (3, 64, 128), (2, 192, 16), (2, 385, 400)])
def test_channels_first_with_odd_numbers_of_pixels(eng, n, pixels, c, dtype):  # noqa: F811
    """Whole tiles (64 pixels of f32, 128 of 16 bits; 256 of the way back) whose channels begin at every second byte of a word, and their ends."""
    from tests.q8_definition import define
    g = torch.Generator().manual_seed(pixels)
    x = (torch.randn(n, pixels, c, generator=g) * torch.exp2(torch.randint(-12, 13, (n, pixels, 1), generator=g).float())).to(dtype)
    x[0, pixels - 1, c - 1], x[n - 1, pixels // 2, 0], x[n - 1, 0, c // 2] = float('nan'), float('inf'), -float('inf')
    codes, scale = define(x.double().view(-1, c).numpy())
    got = eng.quantize(x.permute(0, 2, 1).contiguous().cuda(), channel_major=True)
    assert np.array_equal(got.codes.cpu().double().view(-1, c).numpy(), codes, equal_nan=True)
    assert np.array_equal(got.scale.cpu().double().view(codes.shape[0], -1).numpy(), scale)
    numbers = torch.from_numpy(decode(*got)).view(n, pixels, c)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        back = eng.dequantize(*got, channel_major=True, dtype=out).cpu()
        want = numbers.float().to(out).permute(0, 2, 1)                        # f32 holds the numbers exactly: one rounding
        assert torch.equal(back.isnan(), want.isnan()) and torch.equal(back.nan_to_num(7.0), want.nan_to_num(7.0))

"""The 8-bit feature operators on the GPU against their definition in 64 bits (tests/q8_definition.py).

Tolerances.  Quantising and reading back are exact: x 2^-e and code 2^e are, and the one rounding of either is defined.  A product
of K channels is a sum of K products, each exact in fp32 (8 significant bits at most), added in fp32 in some order: at most
K additions, each off by at most one step relative to a partial sum (2^-23: the matrix cores may cut instead of round), and no partial
sum is larger than S = sum |a_c b_c|.  So |error| <= K 2^-23 S; bf16 results add half a step, 2^-8 of the result.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from nemo_amd import _lib, q8  # noqa: E402
from tests.q8_definition import decode, define, hard_rows  # noqa: E402

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope='module')
def eng():
    from nemo_amd.engine import PoseEngine
    return PoseEngine(24, (12, 23), 128)


def bits(t):
    return t.cpu().view(torch.uint8)


def same_codes(a, b):
    """Equal bits, but for the sign of a NaN."""
    a, b = bits(a), bits(b)
    nan = ((a & 127) == 127) & ((b & 127) == 127)
    return bool(((a == b) | nan).all())


def rows8(rows, k, seed, spread=6):
    """Random rows held in 8 bits, on the GPU, and their numbers in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-spread, spread + 1, (rows, 1), generator=g).float())
    q = q8.quantize_host(x)
    return q8.Q8(q.codes.cuda(), q.scale.cuda()), torch.from_numpy(decode(q.codes, q.scale))


def close(got, a, b, k):
    """got against a b^T (64 bits) within the bound above."""
    want, bound = a @ b.t(), k * 2.0 ** -23 * (a.abs() @ b.abs().t())
    if got.dtype == torch.bfloat16:
        bound = bound * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-300)).max())


# ------------------------------------------------------------------------------------------------ quantise and read back
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('c', [16, 112, 128, 144, 256, 400])
def test_quantize_rows(eng, c, dtype):
    x = hard_rows(257, c, seed=c).to(dtype)
    got = eng.quantize(x.cuda())
    codes, scale = define(x.double().numpy())
    assert np.array_equal(got.codes.cpu().double().numpy(), codes, equal_nan=True)
    assert np.array_equal(got.scale.cpu().double().numpy(), scale)
    back = eng.dequantize(*got)
    with np.errstate(over='ignore'):
        assert np.array_equal(back.cpu().numpy(), decode(got.codes, got.scale).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n,h,w,c', [(1, 1, 1, 128), (3, 12, 23, 128), (2, 5, 13, 256), (4, 7, 9, 48), (2, 8, 8, 208), (1, 1, 63, 16), (2, 13, 5, 384)])
def test_layouts_agree(eng, n, h, w, c, dtype):
    x = hard_rows(max(13, n * h * w), c, seed=n + c)[:n * h * w].reshape(n, h, w, c).to(dtype)
    want = q8.quantize_host(x)
    last = eng.quantize(x.cuda())
    first = eng.quantize(x.permute(0, 3, 1, 2).contiguous().cuda(), channel_major=True)
    for got in (last, first):
        assert got.codes.shape == want.codes.shape and same_codes(got.codes, want.codes)
        assert torch.equal(bits(got.scale), bits(want.scale))
    for out in DTYPES:
        want_x = q8.dequantize_host(want, out)
        a = eng.dequantize(*last, dtype=out)
        b = eng.dequantize(*last, channel_major=True, dtype=out)
        assert a.dtype == b.dtype == out
        assert torch.equal(a.cpu().nan_to_num(7.0), want_x.nan_to_num(7.0)) and torch.equal(a.isnan().cpu(), want_x.isnan())
        assert b.shape == (n, c, h, w) and torch.equal(b.cpu().nan_to_num(7.0), want_x.permute(0, 3, 1, 2).nan_to_num(7.0))


@pytest.mark.parametrize('channel_major', [False, True])
def test_slots(eng, channel_major):
    n, h, w, c, room = 9, 6, 11, 144, 12
    x = torch.randn(n, h, w, c, generator=torch.Generator().manual_seed(3))
    want = q8.quantize_host(x)
    slots = torch.tensor([4, 0, 4, -1, 11, 12, 7, 4, 0], dtype=torch.int32)   # 4 and 0 named again, -1 and 12 outside
    cache = q8.Q8(torch.full((room, h, w, c), 0x55, dtype=torch.uint8).cuda().view(torch.float8_e4m3fn),
                  torch.full((room, h, w, 2), 0x66, dtype=torch.uint8).cuda().view(torch.float8_e8m0fnu))
    src = (x.permute(0, 3, 1, 2).contiguous() if channel_major else x).cuda()
    got = eng.quantize(src, channel_major=channel_major, slots=slots.cuda(), out=cache)
    assert got.codes.data_ptr() == cache.codes.data_ptr()
    last = {4: 7, 0: 8, 11: 4, 7: 6}
    for s in range(room):
        if s in last:
            assert torch.equal(bits(cache.codes[s]), bits(want.codes[last[s]])) and torch.equal(bits(cache.scale[s]), bits(want.scale[last[s]]))
        else:
            assert bool((bits(cache.codes[s]) == 0x55).all()) and bool((bits(cache.scale[s]) == 0x66).all())
    read = torch.tensor([7, 7, 12, 0, -5, 4], dtype=torch.int32)              # twice the same, and two outside
    back = eng.dequantize(*cache, slots=read.cuda(), channel_major=channel_major).cpu()
    for i, s in enumerate(read.tolist()):
        y = q8.dequantize_host(q8.Q8(want.codes[last[s]], want.scale[last[s]])) if s in last else torch.zeros(h, w, c)
        assert torch.equal(back[i], y.permute(2, 0, 1) if channel_major else y)


def test_scale_bytes_at_the_ends(eng):
    codes = torch.arange(256, dtype=torch.uint8).repeat(3, 1).view(torch.float8_e4m3fn)
    scale = torch.tensor([[0, 1], [2, 254], [255, 127]], dtype=torch.uint8).view(torch.float8_e8m0fnu)
    got = eng.dequantize(codes.cuda(), scale.cuda()).cpu().numpy()
    with np.errstate(over='ignore'):
        assert np.array_equal(got, decode(codes, scale).astype(np.float32), equal_nan=True)


def test_offsets_beyond_32_bits(eng):
    rows, c, room = 1 << 20, 1024, 5                                          # 1 GiB of codes an image
    cache = q8.empty((room, rows, c), 'cuda')
    x = torch.randn(1, rows, c, device='cuda', dtype=torch.float16, generator=torch.Generator('cuda').manual_seed(1))
    alone = eng.quantize(x)
    eng.quantize(x, slots=torch.tensor([4], dtype=torch.int32, device='cuda'), out=cache)
    assert torch.equal(cache.codes[4].view(torch.uint8), alone.codes[0].view(torch.uint8))
    assert torch.equal(cache.scale[4].view(torch.uint8), alone.scale[0].view(torch.uint8))
    y = eng.dequantize(*cache, slots=torch.tensor([4], dtype=torch.int32, device='cuda'), dtype=torch.float16)
    assert torch.equal(y, eng.dequantize(*alone, dtype=torch.float16))
    a, b = q8.Q8(cache.codes.view(-1, c), cache.scale.view(-1, c // 128)), eng.quantize(x[0, :3].contiguous())
    seg = torch.tensor([5 * rows - 7, 5 * rows], dtype=torch.int32, device='cuda')
    got = eng.q8_grouped_product(a, seg, b, torch.tensor([0, 3], dtype=torch.int32, device='cuda'))
    want = eng.q8_product(q8.Q8(alone.codes[0, -7:].contiguous(), alone.scale[0, -7:].contiguous()), b)
    assert torch.equal(got[-7:], want) and not bool(got[:-7].any())


# ------------------------------------------------------------------------------------------------ products
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('m,n,k', [(1, 1, 16), (1, 1088, 128), (33, 31, 128), (127, 129, 144), (128, 128, 256), (200, 1, 512), (257, 300, 240),
                                   (1000, 77, 128), (129, 260, 2048), (64, 33, 4112),
                                   (8000, 1088, 128), (33001, 77, 256), (17000, 261, 64), (9001, 1000, 240),
                                   (8200, 129, 1024), (1000, 1030, 400), (5000, 257, 272)])
def test_product(eng, m, n, k, dtype):
    (a, a64), (b, b64) = rows8(m, k, m + k), rows8(n, k, n + k + 1)
    got = eng.q8_product(a, b, dtype=dtype)
    assert got.shape == (m, n) and got.dtype == dtype
    close(got, a64, b64, k)


def test_product_of_maps_and_empty_ones(eng):
    (a, a64), (b, b64) = rows8(2 * 3 * 5, 128, 1), rows8(9, 128, 2)
    a4 = q8.Q8(a.codes.view(2, 3, 5, 128), a.scale.view(2, 3, 5, 1))
    got = eng.q8_product(a4, b)
    assert got.shape == (2, 3, 5, 9)
    close(got.view(30, 9), a64, b64, 128)
    none = q8.empty((0, 128), 'cuda')
    assert eng.q8_product(none, b).shape == (0, 9) and eng.q8_product(b, none).shape == (9, 0)
    assert eng.quantize(torch.empty(0, 128, device='cuda')).codes.shape == (0, 128)
    assert eng.dequantize(*none).shape == (0, 128)


def test_product_nan_stays_in_its_row_and_column(eng):
    (a, a64), (b, b64) = rows8(70, 256, 5), rows8(40, 256, 6)
    a.codes.view(torch.uint8)[13, 200] = 0x7f
    b.codes.view(torch.uint8)[39, 0] = 0xff
    got = eng.q8_product(a, b).cpu()
    want = torch.zeros(70, 40, dtype=torch.bool)
    want[13], want[:, 39] = True, True
    assert torch.equal(got.isnan(), want)


def test_scales_of_any_size_meet_exactly(eng):
    """Rows of 2^-100 times rows of 2^100: the scales multiply, nothing overflows on the way."""
    (a, a64), (b, b64) = rows8(50, 128, 7, spread=0), rows8(60, 128, 8, spread=0)
    a = q8.Q8(a.codes, (a.scale.view(torch.uint8) - 100).view(torch.float8_e8m0fnu))
    b = q8.Q8(b.codes, (b.scale.view(torch.uint8) + 100).view(torch.float8_e8m0fnu))
    close(eng.q8_product(a, b), a64 * 2.0 ** -100, b64 * 2.0 ** 100, 128)


@pytest.mark.parametrize('k', [128, 256, 1024])
def test_scale_bytes_at_the_ends_in_products(eng, k):
    """Byte 255 stands for NaN wherever the row is used; the smallest scales, 2^-127 among them, multiply with large ones."""
    (a, a64), (b, b64) = rows8(300, k, 9, spread=0), rows8(300, k, 10, spread=0)
    a.scale.view(torch.uint8)[7, -1] = 255
    b.scale.view(torch.uint8)[299, 0] = 255
    got = eng.q8_product(a, b).cpu()
    want = torch.zeros(300, 300, dtype=torch.bool)
    want[7], want[:, 299] = True, True
    assert torch.equal(got.isnan(), want)
    (a, _), (b, _) = rows8(300, k, 11, spread=0), rows8(40, k, 12, spread=0)
    for byte in (0, 1, 2, 5):
        low = q8.Q8(a.codes, torch.full_like(a.scale.view(torch.uint8), byte).view(torch.float8_e8m0fnu))
        high = q8.Q8(b.codes, torch.full_like(b.scale.view(torch.uint8), 240).view(torch.float8_e8m0fnu))
        close(eng.q8_product(low, high), torch.from_numpy(decode(*low)), torch.from_numpy(decode(*high)), k)


def offsets(sizes):
    return torch.tensor([0] + list(np.cumsum(sizes)), dtype=torch.int32).cuda()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('sizes,banks,bank_of,k', [
    ([5], [7], None, 128),
    ([0, 130, 1, 0, 257, 3], [40, 1, 0, 33, 300, 64], None, 128),
    ([64, 64, 200], [130], None, 256),
    ([31, 129, 7, 100], [50, 160, 20], [2, 0, 5, 0], 144),
    ([300, 2, 0, 5], [10, 1], [1, 0, 1, -1], 512),
    ([5000, 300, 20000, 7, 0, 8000], [300, 500, 129, 1000, 3, 1], None, 128),
    ([9000, 8500, 300], [1, 515], [1, 1, 0], 256),
    ([12000, 5000], [130, 700], None, 80),
    ([3000, 129, 0, 2500], [260, 1, 20, 300], [0, 3, 1, 2], 528),
    ([(i * 37) % 90 for i in range(700)], [(i * 13) % 41 for i in range(700)], None, 128),
])
def test_grouped_product(eng, sizes, banks, bank_of, k, dtype):
    behind = 11                                                               # rows and bank rows of no segment and no bank
    (a, a64), (b, b64) = rows8(sum(sizes) + behind, k, 11), rows8(sum(banks) + behind, k, 12)
    cols = max(banks) + 3
    out = torch.full((sum(sizes) + behind, cols), 123.0, dtype=dtype, device='cuda')
    of = None if bank_of is None else torch.tensor(bank_of, dtype=torch.int32).cuda()
    got = eng.q8_grouped_product(a, offsets(sizes), b, offsets(banks), bank_of=of, out=out)
    assert got.data_ptr() == out.data_ptr()
    left = torch.ones(out.shape, dtype=torch.bool)
    m0, starts = 0, np.cumsum([0] + banks)
    for s, m in enumerate(sizes):
        g = bank_of[s] if bank_of is not None else 0 if len(banks) == 1 else s
        if 0 <= g < len(banks):
            n0, n1 = int(starts[g]), int(starts[g + 1])
            close(out[m0:m0 + m, :n1 - n0], a64[m0:m0 + m], b64[n0:n1], k)
            left[m0:m0 + m, :n1 - n0] = False
        m0 += m
    assert bool((out.cpu()[left] == 123.0).all())
    if bank_of is None and len(banks) > 1:                                    # fewer columns than a bank has rows
        few = eng.q8_grouped_product(a, offsets(sizes), b, offsets(banks), n_cols=9, dtype=dtype)
        m0 = 0
        for m, n in zip(sizes, banks):
            assert torch.equal(few[m0:m0 + m, :min(n, 9)], out[m0:m0 + m, :min(n, 9)])
            m0 += m


def test_grouped_rows_do_not_depend_on_their_company(eng):
    """A row's products are the same bits alone, in a group and in one large product."""
    (a, _), (b, _) = rows8(500, 256, 21), rows8(90, 256, 22)
    whole = eng.q8_product(a, b)
    cut = eng.q8_grouped_product(a, offsets([3, 0, 130, 200, 167]), b, offsets([90]), n_cols=90)
    one = eng.q8_product(q8.Q8(a.codes[77:78].contiguous(), a.scale[77:78].contiguous()), b)
    assert torch.equal(whole, cut) and torch.equal(whole[77:78], one)


def score64(a64, b64):
    return (a64 @ b64.t()).max(1).values if len(b64) else torch.full((len(a64),), -math.inf, dtype=torch.float64)


@pytest.mark.parametrize('d', [128, 256])
@pytest.mark.parametrize('n,h,w,banks', [(1, 12, 23, [1]), (3, 5, 7, [64]), (5, 8, 16, [33, 0, 1, 200]), (2, 1, 1, [2560]), (7, 9, 31, [5, 17, 31, 32, 96, 513]),
                                         (260, 5, 7, [33, 0, 1, 200, 130]), (130, 24, 30, [129, 40]), (130, 15, 20, [300, 1, 31])])
def test_clutter_score(n, h, w, banks, d):
    from nemo_amd.engine import PoseEngine
    eng = PoseEngine(max(h, w, 24), (h, w), d)
    (a, a64), (b, b64) = rows8(n * h * w, d, 31 + n), rows8(sum(banks), d, 32)
    a = q8.Q8(a.codes.view(n, h, w, d), a.scale.view(n, h, w, d // 128))
    a64 = a64.view(n, h * w, d)
    of = [(3 * i + 1) % len(banks) for i in range(n)]
    starts = np.cumsum([0] + banks)   # (the last three: enough tiles of 1024, 512 and 256 pixels to fill the GPU with them)
    out = torch.full((n, h, w), 5.0, device='cuda')
    index = torch.tensor(of, dtype=torch.int32)
    if n > 2:
        index[n - 1] = len(banks)                                             # no such bank: left as it was
    got = eng.q8_clutter_score(a, b, offsets(banks), index.cuda(), out=out)
    for i in range(n):
        g = of[i]
        rows = b64[int(starts[g]):int(starts[g + 1])]
        if index[i] == len(banks):
            assert bool((got[i] == 5.0).all())
        elif len(rows) == 0:
            assert bool((got[i] == -math.inf).all())
        else:
            bound = d * 2.0 ** -23 * (a64[i].abs() @ rows.abs().t()).max(1).values   # the maximum moves no further than its terms
            assert bool(((got[i].cpu().double().view(-1) - score64(a64[i], rows)).abs() <= bound).all())
    whole = eng.q8_clutter_score(a, b)                                        # all rows one bank
    bound = d * 2.0 ** -23 * (a64.abs() @ b64.abs().t()).max(2).values
    assert bool(((whole.cpu().double().view(n, -1) - (a64 @ b64.t()).max(2).values).abs() <= bound).all())


def test_clutter_score_nan(eng):
    (a, _), (b, _) = rows8(2 * 12 * 23, 128, 41), rows8(70, 128, 42)
    a = q8.Q8(a.codes.view(2, 12, 23, 128), a.scale.view(2, 12, 23, 1))
    a.codes.view(torch.uint8)[1, 3, 4, 5] = 0x7f
    got = eng.q8_clutter_score(a, b).cpu()
    assert bool(got[1, 3, 4].isnan()) and int(got.isnan().sum()) == 1
    b.codes.view(torch.uint8)[69, 127] = 0x7f
    assert bool(eng.q8_clutter_score(a, b).isnan().all())
    (b, _) = rows8(70, 128, 42)
    b.scale.view(torch.uint8)[0, 0] = 255
    assert bool(eng.q8_clutter_score(a, b).isnan().all())


def test_clutter_score_against_the_f32_one(eng):
    """On the numbers the 8-bit maps stand for, nemo_clutter_score gives the same scores."""
    (a, a64), (b, b64) = rows8(3 * 12 * 23, 128, 51, spread=0), rows8(90, 128, 52, spread=0)
    a = q8.Q8(a.codes.view(3, 12, 23, 128), a.scale.view(3, 12, 23, 1))
    got, f32 = eng.q8_clutter_score(a, b), eng.clutter_score(eng.dequantize(*a), eng.dequantize(*b))
    bound = 2 * 128 * 2.0 ** -23 * (a64.abs() @ b64.abs().t()).max(1).values.view(3, 12, 23)   # either side's
    assert bool(((got - f32).cpu().double().abs() <= bound).all())


# ------------------------------------------------------------------------------------------------ as they are called
def chain(eng, x, b, slots, off, of, buf):
    eng.quantize(x, channel_major=True, slots=slots, out=buf['cache'])
    eng.q8_clutter_score(buf['cache'], b, off, of, out=buf['score'])
    eng.dequantize(*buf['cache'], slots=slots, out=buf['back'])
    eng.q8_product(buf['cache'], b, out=buf['all'])
    eng.q8_grouped_product(buf['rows'], buf['row_off'], b, off, bank_of=of, out=buf['grouped'])


def buffers(n, h, w, c, k):
    cache = q8.Q8(torch.zeros(n, h, w, c, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn),
                  torch.zeros(n, h, w, c // 128, dtype=torch.uint8, device='cuda').view(torch.float8_e8m0fnu))
    return {'cache': cache, 'score': torch.zeros(n, h, w, device='cuda'), 'back': torch.zeros(n, h, w, c, device='cuda'),
            'all': torch.zeros(n, h, w, k, device='cuda'), 'grouped': torch.zeros(n * h * w, k, device='cuda'),
            'rows': q8.Q8(cache.codes.view(-1, c), cache.scale.view(n * h * w, -1)), 'row_off': offsets([h * w] * n)}


def test_captured_chain_replays(eng):
    n, h, w, c, k = 4, 12, 23, 128, 75
    (b, _) = rows8(k, c, 61)
    slots, of, off = torch.tensor([2, 0, 3, 1], dtype=torch.int32).cuda(), torch.tensor([0, 1, 1, 0], dtype=torch.int32).cuda(), offsets([40, 35])
    x = torch.zeros(n, c, h, w, device='cuda')
    buf, ref = buffers(n, h, w, c, k), buffers(n, h, w, c, k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(eng, x, b, slots, off, of, buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(eng, x, b, slots, off, of, buf)
    for seed in range(4):
        x.copy_(torch.randn(n, c, h, w, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        chain(eng, x.clone(), b, slots, off, of, ref)                         # eager work between the replays
        torch.cuda.synchronize()
        for key in ('score', 'back', 'all', 'grouped'):
            assert torch.equal(buf[key], ref[key]) and bool(buf[key].any()), (seed, key)


def test_two_streams_at_once(eng):
    n, h, w, c, k = 6, 12, 23, 128, 200
    (b, _) = rows8(k, c, 71)
    slots, of, off = torch.arange(n, dtype=torch.int32).cuda(), (torch.arange(n) % 2).int().cuda(), offsets([150, 50])
    xs = [torch.randn(n, c, h, w, generator=torch.Generator().manual_seed(s)).cuda() for s in range(2)]
    want, got, streams = [buffers(n, h, w, c, k) for _ in xs], [buffers(n, h, w, c, k) for _ in xs], [torch.cuda.Stream() for _ in xs]
    for x, buf in zip(xs, want):
        chain(eng, x, b, slots, off, of, buf)
    torch.cuda.synchronize()
    for _ in range(5):
        for x, buf, s in zip(xs, got, streams):
            with torch.cuda.stream(s):
                chain(eng, x, b, slots, off, of, buf)
    torch.cuda.synchronize()
    for a, b_ in zip(want, got):
        for key in ('score', 'back', 'all', 'grouped'):
            assert torch.equal(a[key], b_[key]), key


def test_same_result_every_time(eng):
    (a, _), (b, _) = rows8(12 * 23 * 5, 128, 81), rows8(700, 128, 82)
    a = q8.Q8(a.codes.view(5, 12, 23, 128), a.scale.view(5, 12, 23, 1))
    first = eng.q8_clutter_score(a, b), eng.q8_product(a, b)
    for _ in range(3):
        assert torch.equal(eng.q8_clutter_score(a, b), first[0]) and torch.equal(eng.q8_product(a, b), first[1])


# ------------------------------------------------------------------------------------------------ in the solver
def test_solver_on_maps_in_8_bits():
    """BatchPoseSolver on 8-bit maps is the solver on the numbers they stand for, bit for bit, with the 8-bit clutter scores."""
    from nemo_amd.pose_solver import SolverConfig
    from nemo_amd.workloads import twelve_class_workload
    wl = twelve_class_workload(10, seed=5, cfg=SolverConfig(image_size=(256, 384), total_epochs=20), categories=['car', 'sofa', 'chair'])
    s, eng = wl.solver, wl.solver.engine
    maps = eng.quantize(wl.feats)
    back = eng.dequantize(*maps)
    # every number within half a step of its code: 2^-4 of it, or 2^-10 of the scale
    step = torch.maximum(wl.feats.abs() * 2.0 ** -4, maps.scale.float() * 2.0 ** -10)
    assert bool(((back - wl.feats).abs() <= step).all())
    group = [int(m) for m in wl.mesh_idx]
    rng = torch.Generator().manual_seed(1)
    clutter = [torch.nn.functional.normalize(torch.randn(k, 128, generator=rng)).cuda() for k in (1, 7, 40)]
    banks = s.clutter_banks8(clutter)
    clu = s.clutter_scores_by_group(maps, group, banks)
    assert torch.equal(clu, s.clutter_scores_by_group(maps, group, clutter))
    for i, g in enumerate(group):                          # alone, each image against its own bank
        one = q8.Q8(maps.codes[i:i + 1].contiguous(), maps.scale[i:i + 1].contiguous())
        assert torch.equal(clu[i], eng.q8_clutter_score(one, eng.quantize(clutter[g]))[0])
    a = s.solve_all(maps, None, wl.mesh_idx, clutter_scores=clu)
    b = s.solve_all(back, None, wl.mesh_idx, clutter_scores=clu)
    assert torch.equal(a.campos, b.campos) and torch.equal(a.loss, b.loss) and torch.equal(a.init_index, b.init_index)
    c = s.solve_all(maps, wl.clutter, wl.mesh_idx)          # one clutter vector for all
    d = s.solve_all(back, None, wl.mesh_idx, clutter_scores=eng.q8_clutter_score(maps, eng.quantize(wl.clutter)))
    assert torch.equal(c.campos, d.campos) and torch.equal(c.loss, d.loss) and bool(torch.isfinite(c.loss).all())
    with pytest.raises(ValueError, match='group_of_image'):
        s.clutter_scores_by_group(maps, [0] * 9 + [3], banks)
    with pytest.raises(ValueError, match='at least one clutter vector'):
        s.clutter_banks8([clutter[0], clutter[1][:0]])


def test_runner_on_a_record_in_8_bits(tmp_path):
    """The file-driven runner on an 8-bit record: the solver on the record's numbers, in batches on two streams."""
    from nemo_amd import mesh_utils, records, solve_all
    from nemo_amd import synthetic as syn
    rng = np.random.default_rng(3)
    names, feats, mem, clu = {}, {}, {}, {}
    for k, st in enumerate(('mesh01', 'mesh02')):
        v, f = syn.class_mesh('car', 300 + 50 * k)
        mesh_utils.save_off(str(tmp_path / ('%02d.off' % (k + 1))), v, f)
        mem[st], clu[st] = syn.unit_rows(rng, len(v), 128), syn.unit_rows(rng, 6 + k, 128)
        names[st] = ['%s_%d' % (st, i) for i in range(11)]
        for n in names[st]:
            feats[n] = syn.unit_rows(rng, 12 * 23, 128).reshape(12, 23, 128).transpose(2, 0, 1).copy()
    src, dst = str(tmp_path / 'f32.npz'), str(tmp_path / 'q8.npz')
    records.write_feature_record(src, mem, clu, names, feats)
    records.quantize_record(src, dst)
    args = solve_all.build_parser().parse_args(['--type_', 'car', '--record_file', dst, '--mesh_path', str(tmp_path), '--image_size', '96,184',
                                                '--total_epochs', '15', '--batch', '8'])
    with records.FeatureRecord(dst) as rec:
        all_names, mesh_of = solve_all.category_jobs(rec, ['mesh01', 'mesh02'])
        order = [i for pair in zip(range(11), range(11, 22)) for i in pair]   # the subtypes in turn
        all_names, mesh_of = [all_names[i] for i in order], [mesh_of[i] for i in order]
        got, _ = solve_all.solve_shard(args, rec, ['mesh01', 'mesh02'], all_names, mesh_of, 'cuda:0')
        maps = rec.upload8(all_names, 'cuda:0', chunk=5)
        assert torch.equal(rec.upload_pixel_major(all_names, 'cuda:0').cpu(),
                           torch.stack([torch.from_numpy(rec.feature(n)).permute(1, 2, 0) for n in all_names]))
        solver, clutter = solve_all.build_solver(args, rec, ['mesh01', 'mesh02'], 'cuda:0')
        mesh = torch.tensor(mesh_of, dtype=torch.int32, device='cuda')
        want = solver.solve_all(solver.engine.dequantize(*maps), None, mesh, clutter_scores=solver.clutter_scores_by_group(maps, mesh_of, clutter))
    assert torch.equal(got[:, :8], want.packed())


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(eng):
    (a, _), (b, _) = rows8(12 * 23, 128, 91), rows8(8, 128, 92)
    maps = q8.Q8(a.codes.view(1, 12, 23, 128), a.scale.view(1, 12, 23, 1))
    x = torch.zeros(1, 12, 23, 128, device='cuda')
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device='cuda')  # noqa: E731
    for error, call in [
        (TypeError, lambda: eng.quantize(x.double())),
        (ValueError, lambda: eng.quantize(x.cpu())),
        (ValueError, lambda: eng.quantize(x.transpose(1, 2))),
        (ValueError, lambda: eng.quantize(x[0, 0, 0])),
        (ValueError, lambda: eng.quantize(x, slots=i32(0))),
        (ValueError, lambda: eng.quantize(x, slots=i32(0, 1), out=maps)),
        (TypeError, lambda: eng.quantize(x, slots=i32(0).long(), out=maps)),
        (ValueError, lambda: eng.quantize(x, out=q8.empty((1, 12, 22, 128), 'cuda'))),
        (ValueError, lambda: eng.quantize(x, out=q8.empty((2, 12, 23, 128), 'cuda'))),
        (_lib.NemoHipError, lambda: eng.quantize(torch.zeros(4, 24, device='cuda'))),
        (_lib.NemoHipError, lambda: eng.quantize(torch.zeros(4 * 128 + 1, device='cuda')[1:].view(4, 128))),
        (TypeError, lambda: eng.dequantize(a.codes.view(torch.uint8), a.scale)),
        (TypeError, lambda: eng.dequantize(*maps, slots=[0])),
        (ValueError, lambda: eng.dequantize(a.codes, a.scale[:-1])),
        (TypeError, lambda: eng.dequantize(a.codes, a.scale, dtype=torch.float64)),
        (ValueError, lambda: eng.dequantize(*a, channel_major=True)),
        (ValueError, lambda: eng.dequantize(*maps, out=torch.zeros(1, 128, 12, 23, device='cuda'))),
        (ValueError, lambda: eng.q8_product(a, rows8(8, 256, 1)[0])),
        (ValueError, lambda: eng.q8_product(a, maps)),
        (TypeError, lambda: eng.q8_product(a, b, dtype=torch.float16)),
        (ValueError, lambda: eng.q8_product(a, b, out=torch.zeros(8, 276, device='cuda'))),
        (ValueError, lambda: eng.q8_grouped_product(maps, i32(0, 1), b, i32(0, 8))),
        (ValueError, lambda: eng.q8_grouped_product(a, None, b, i32(0, 8))),
        (TypeError, lambda: eng.q8_grouped_product(a, i32(0, 1).long(), b, i32(0, 8))),
        (ValueError, lambda: eng.q8_grouped_product(a, i32(0, 1), b, i32(0, 8), bank_of=i32(0, 0))),
        (_lib.NemoHipError, lambda: eng.q8_grouped_product(a, i32(0, 1, 2, 3), b, i32(0, 4, 8))),
        (ValueError, lambda: eng.q8_clutter_score(a, b)),
        (ValueError, lambda: eng.q8_clutter_score(maps, maps)),
        (ValueError, lambda: eng.q8_clutter_score(maps, rows8(8, 256, 1)[0])),
        (ValueError, lambda: eng.q8_clutter_score(maps, b, i32(0, 4, 8), i32(0, 1))),
        (_lib.NemoHipError, lambda: eng.q8_clutter_score(maps, b, i32(0, 2, 4, 8))),
        (TypeError, lambda: eng.q8_clutter_score(maps, b, out=torch.zeros(1, 12, 23, device='cuda', dtype=torch.bfloat16))),
    ]:
        with pytest.raises(error):
            call()
    assert torch.equal(eng.q8_product(a, b), eng.q8_product(a, b))            # still usable


def test_validated_indices():
    from nemo_amd.engine import PoseEngine
    eng = PoseEngine(24, (12, 23), 128, validate_indices=True)
    (a, _), (b, _) = rows8(12 * 23, 128, 91), rows8(8, 128, 92)
    maps = q8.Q8(a.codes.view(1, 12, 23, 128), a.scale.view(1, 12, 23, 1))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device='cuda')  # noqa: E731
    for call in (lambda: eng.quantize(torch.zeros(1, 12, 23, 128, device='cuda'), slots=i32(1), out=maps),
                 lambda: eng.dequantize(*maps, slots=i32(-1)),
                 lambda: eng.q8_grouped_product(a, i32(0, 300), b, i32(0, 8)),
                 lambda: eng.q8_grouped_product(a, i32(0, 5, 3), b, i32(0, 4, 8)),
                 lambda: eng.q8_grouped_product(a, i32(0, 5), b, i32(0, 9)),
                 lambda: eng.q8_clutter_score(maps, b, i32(0, 8), i32(1))):
        with pytest.raises(ValueError):
            call()

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


# ------------------------------------------------------------------------------------------------ records held in 8 bits
def _record(tmp_path, n=7, D=128, h=5, w=9):
    from nemo_amd import records
    rng = np.random.default_rng(4)
    feats = {'img%d' % i: rng.standard_normal((D, h, w)).astype(np.float32) for i in range(n)}
    bank = rng.standard_normal((11, D)).astype(np.float32)
    path = str(tmp_path / 'f32.npz')
    records.write_feature_record(path, {'mesh01': bank}, {'mesh01': bank[:4]}, {'mesh01': list(feats)}, feats)
    return path, feats, bank


@pytest.mark.parametrize('compressed', [False, True])
def test_record_in_8_bits(tmp_path, compressed):
    from nemo_amd import records
    src, feats, bank = _record(tmp_path)
    dst = str(tmp_path / 'q8.npz')
    assert records.quantize_record(src, dst) == len(feats)
    if compressed:
        with np.load(dst) as z:
            np.savez_compressed(dst, **{k: z[k] for k in z.files})
    want = {n: q8.quantize_host(torch.from_numpy(f.transpose(1, 2, 0).copy())) for n, f in feats.items()}
    with records.FeatureRecord(dst) as r:
        assert r.shape8 == (5, 9, 128) and r.feature_shape('img2') == (128, 5, 9) and sorted(r.image_keys) == sorted(feats)
        assert np.array_equal(r.memory('mesh01'), bank) and np.array_equal(r.clutter('mesh01'), bank[:4]) and r.names('mesh01') == list(feats)
        back = q8.dequantize_host(want['img3']).permute(2, 0, 1).numpy()
        assert np.array_equal(r.feature('img3'), back)
        into = np.empty((128, 5, 9), np.float32)
        r.read_feature_into('img3', into)
        assert np.array_equal(into, back)
        for chunk, workers in ((2, 3), (64, 1)):
            st = {}
            got = r.upload8(list(feats), 'cpu', chunk=chunk, workers=workers, stats=st)
            assert got.codes.shape == (7, 5, 9, 128) and st['bytes'] == 7 * 45 * 129
            for i, n in enumerate(feats):
                assert torch.equal(got.codes[i].view(torch.uint8), want[n].codes.view(torch.uint8))
                assert torch.equal(got.scale[i].view(torch.uint8), want[n].scale.view(torch.uint8))
        maps = r.upload_pixel_major(['img5', 'img0'], 'cpu')
        assert torch.equal(maps[0], q8.dequantize_host(want['img5'])) and torch.equal(maps[1], q8.dequantize_host(want['img0']))
    with records.FeatureRecord(src) as r:
        assert r.shape8 is None
        with pytest.raises(ValueError, match='not held in 8 bits'):
            r.upload8(['img0'], 'cpu')
        with pytest.raises(ValueError, match='not held in 8 bits'):
            r.feature8('img0')


def test_record_in_8_bits_refusals(tmp_path):
    from nemo_amd import records
    src, feats, bank = _record(tmp_path, n=2)
    dst = str(tmp_path / 'q8.npz')
    with pytest.raises(ValueError, match='overwrite its source'):
        records.quantize_record(src, src)
    records.quantize_record(src, dst)
    with pytest.raises(ValueError, match='in 8 bits already'):
        records.quantize_record(dst, str(tmp_path / 'again.npz'))
    a, b = q8.quantize_host(torch.zeros(5, 9, 128)), q8.quantize_host(torch.zeros(5, 8, 128))
    with pytest.raises(ValueError, match='of one shape'):
        records.write_feature_record8(dst, {}, {}, {}, {'a': a, 'b': b})
    with pytest.raises(ValueError, match='no feature maps'):
        records.write_feature_record8(dst, {}, {}, {}, {})
    np.savez(dst, features_8bit=np.array([5, 9, 128]), img=np.zeros(17, np.uint8))
    with records.FeatureRecord(dst) as r:
        with pytest.raises(ValueError, match='expected %d bytes' % (45 * 129)):
            r.feature8('img')
        with pytest.raises(ValueError, match='expected %d bytes' % (45 * 129)):
            r.upload8(['img'], 'cpu')


def test_runner_writes_a_record_in_8_bits(tmp_path, capsys):
    from nemo_amd import records, solve_all
    src, feats, _ = _record(tmp_path)
    dst = str(tmp_path / 'sub' / 'q8.npz')
    assert solve_all.main(['--type_', 'car', '--record_file', src, '--quantize_record', dst]) == 0
    assert '7 maps in 8 bits' in capsys.readouterr().out
    with records.FeatureRecord(dst) as r:
        assert r.shape8 == (5, 9, 128)


def test_record_used_again_after_close_and_with_long_names(tmp_path):
    """Layouts are found again after close(), for members with other headers and for names longer than what is read of a header at once."""
    from nemo_amd import records
    long = 'x' * 2000
    path = str(tmp_path / 'r.npz')
    a, b, c = (np.arange(n * 20, dtype=np.float32).reshape(n, 4, 5) for n in (3, 30, 300))
    np.savez(path, **{'a': a, 'b': b, 'c': c, long: 2 * a, long + 'y': 3 * b, 'f16': a.astype(np.float16), 'fortran': np.asfortranarray(b)})
    r = records.FeatureRecord(path)
    for _ in range(2):
        for name, want in (('a', a), (long, 2 * a), ('b', b), (long + 'y', 3 * b), ('c', c), ('a', a)):
            into = np.empty_like(want)
            r.read_feature_into(name, into)
            assert np.array_equal(into, want) and r._layout(name)[1] == want.shape
        assert r._layout('f16') is None and r._layout('fortran') is None
        r.close()


def test_runner_writes_the_record_once(tmp_path, monkeypatch):
    from nemo_amd import solve_all
    src, _, _ = _record(tmp_path, n=2)
    dst = tmp_path / 'q8.npz'
    monkeypatch.setenv('RANK', '1')
    assert solve_all.main(['--type_', 'car', '--record_file', src, '--quantize_record', str(dst)]) == 0
    assert not dst.exists()

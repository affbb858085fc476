"""Feature records held in 8 bits: the file that is written, and the one that is read."""
import os
import threading
import time
import zipfile
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from nemo_amd import q8, records, solve_all
from tests.test_q8_cpu import _record


@pytest.mark.parametrize('kind', ['same', 'no suffix', 'symlink', 'symlink without suffix', 'link to the folder', 'hard link', 'relative'])
def test_quantize_record_keeps_its_source(tmp_path, monkeypatch, kind):
    src, feats, _ = _record(tmp_path, n=3)
    assert src.endswith('f32.npz')
    dst = {'same': src, 'no suffix': src[:-4], 'relative': 'f32', 'link to the folder': str(tmp_path / 'sub' / 'f32.npz')}.get(kind, str(tmp_path / 'link.npz'))
    if kind.startswith('symlink'):
        os.symlink(src, dst)
    if kind == 'symlink without suffix':
        dst = dst[:-4]
    if kind == 'link to the folder':
        os.symlink(str(tmp_path), str(tmp_path / 'sub'))
    if kind == 'hard link':
        os.link(src, dst)
    monkeypatch.chdir(tmp_path)
    before, listed = open(src, 'rb').read(), sorted(os.listdir(tmp_path))
    with pytest.raises(ValueError, match='overwrite its source'):
        records.quantize_record(src, dst)
    with pytest.raises(ValueError, match='overwrite its source'):
        solve_all.main(['--type_', 'car', '--record_file', src, '--quantize_record', dst])
    assert open(src, 'rb').read() == before and sorted(os.listdir(tmp_path)) == listed


def test_record_file_is_named_and_read(tmp_path, capsys):
    src, feats, _ = _record(tmp_path, n=3)
    assert solve_all.main(['--type_', 'car', '--record_file', src, '--quantize_record', str(tmp_path / 'q8')]) == 0
    file = str(tmp_path / 'q8.npz')
    assert file in capsys.readouterr().out
    with records.FeatureRecord(file) as r:
        assert r.shape8 == (5, 9, 128) and sorted(r.image_keys) == sorted(feats)


def test_record_is_written_whole_or_not_at_all(tmp_path, monkeypatch):
    src, _, _ = _record(tmp_path, n=3)
    dst = tmp_path / 'q8.npz'
    records.quantize_record(src, str(dst))
    before = dst.read_bytes()

    def fails(fh, **arrays):
        fh.write(b'half')
        raise OSError('no space')
    with monkeypatch.context() as m:
        m.setattr(np, 'savez', fails)
        with pytest.raises(OSError, match='no space'):
            records.quantize_record(src, str(dst))
    assert dst.read_bytes() == before and sorted(os.listdir(tmp_path)) == ['f32.npz', 'q8.npz']
    os.symlink(str(dst), str(tmp_path / 'name.npz'))          # a link to another file: that file is written
    records.write_feature_record8(tmp_path / 'name', {}, {}, {}, {'a': q8.quantize_host(torch.ones(2, 3, 128))})
    with records.FeatureRecord(str(dst)) as r:
        assert r.shape8 == (2, 3, 128)
    assert os.path.islink(tmp_path / 'name.npz')


def test_an_image_may_be_named_like_the_mark(tmp_path):
    """A map called features_8bit in an f32 record is an image; a record in 8 bits cannot hold it."""
    rng = np.random.default_rng(1)
    feats = {n: rng.standard_normal((128, 4, 5)).astype(np.float32) for n in ('a', 'features_8bit')}
    src, dst = str(tmp_path / 'f32.npz'), tmp_path / 'q8.npz'
    records.write_feature_record(src, {}, {}, {}, feats)
    with records.FeatureRecord(src) as r:
        assert r.shape8 is None and sorted(r.image_keys) == sorted(feats) and r.feature_shape('features_8bit') == (128, 4, 5)
        assert all(np.array_equal(r.feature(n), f) for n, f in feats.items())
        got = r.upload_pixel_major(['features_8bit', 'a'], 'cpu')
        assert np.array_equal(got[0].numpy(), feats['features_8bit'].transpose(1, 2, 0))
    with pytest.raises(ValueError, match='cannot be named'):
        records.quantize_record(src, str(dst))
    assert not dst.exists()
    for mark in (np.array([5, 9]), np.array([5, 0, 128]), np.array([5.0, 9.0, 128.0]), np.int64(3)):
        np.savez(dst, features_8bit=mark)
        with pytest.raises(ValueError, match='is not'):
            records.FeatureRecord(str(dst))


def open_files():
    return len(os.listdir('/proc/self/fd'))


def test_directory_of_a_record_leaves_no_file_open(tmp_path, monkeypatch):
    """Asked for at once by several threads, or in vain: one descriptor at most, none after close."""
    src, feats, _ = _record(tmp_path, n=3)
    before = open_files()
    r = records.FeatureRecord(src)
    kept = open_files()
    wait, real = threading.Barrier(8), zipfile.ZipFile

    def slow(*a, **k):
        time.sleep(0.05)
        return real(*a, **k)
    monkeypatch.setattr(records.zipfile, 'ZipFile', slow)

    def ask(name):
        wait.wait()
        return r._layout(name)
    with ThreadPoolExecutor(8) as pool:
        got = list(pool.map(ask, ['img%d' % (i % 3) for i in range(8)]))
    assert all(g[1] == (128, 5, 9) for g in got) and got[0] == got[3] == got[6] != got[1]
    assert open_files() == kept + 1
    r.close()
    assert open_files() == before
    r = records.FeatureRecord(src)

    def broken(*a, **k):
        raise zipfile.BadZipFile('no directory')
    monkeypatch.setattr(records.zipfile, 'ZipFile', broken)
    for _ in range(3):
        with pytest.raises(zipfile.BadZipFile):
            r._layout('img0')
    assert open_files() == kept
    r.close()
    assert open_files() == before


def test_record_takes_and_fills_what_it_names(tmp_path):
    """Maps of other types are not written as if they were codes, and buffers that a read would not reach are refused."""
    a = q8.quantize_host(torch.ones(4, 5, 128))
    dst = tmp_path / 'q8.npz'
    for bad in (q8.Q8(a.codes.float(), a.scale), q8.Q8(a.codes, a.scale.float()), q8.Q8(a.codes.view(torch.uint8), a.scale.view(torch.uint8))):
        with pytest.raises(ValueError, match='expected codes and scales'):
            records.write_feature_record8(str(dst), {}, {}, {}, {'a': bad})
    assert not dst.exists()
    records.write_feature_record8(str(dst), {}, {}, {}, {'a': a})
    codes, scale = np.zeros((4, 5, 128), np.uint8), np.zeros((4, 5, 1), np.uint8)
    with records.FeatureRecord(str(dst)) as r, open(dst, 'rb') as fh:
        r.read_feature8_into('a', codes, scale, fh.fileno())
        assert np.array_equal(codes, a.codes.view(torch.uint8).numpy()) and np.array_equal(scale, a.scale.view(torch.uint8).numpy())
        for c, s in ((codes.transpose(1, 0, 2), scale), (codes[:, ::2], scale), (codes.view(np.int8), scale), (codes[:3], np.zeros((4, 5, 33), np.uint8)),
                     (codes, scale[:, :, [0, 0]]), (codes, np.zeros((4, 5), np.float32))):
            with pytest.raises(ValueError, match='contiguous bytes'):
                r.read_feature8_into('a', c, s, fh.fileno())

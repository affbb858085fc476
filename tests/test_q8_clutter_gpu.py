"""Maps held in 8 bits against clutter vectors that stay f32: only what the caller chose is rounded.

Tolerance of a score: the largest of products of D numbers, each exact or rounded once in fp32 and added in fp32 in some order, is off by
at most (D + 1) 2^-23 sum |f_c c_c| (a step per operation: the matrix cores may cut instead of round).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from nemo_amd import mesh_utils, q8, records, solve_all  # noqa: E402
from nemo_amd import synthetic as syn  # noqa: E402
from tests.q8_definition import decode  # noqa: E402


def scores64(maps, clutter):
    """Scores in 64 bits of the numbers the maps stand for, and the bound above."""
    f = torch.from_numpy(decode(maps.codes, maps.scale))
    c = clutter.cpu().double()
    return (f @ c.t()).amax(-1), (f.shape[-1] + 1) * 2.0 ** -23 * (f.abs() @ c.abs().t()).amax(-1)


def test_solver_with_clutter_vectors_in_f32():
    from nemo_amd.pose_solver import SolverConfig
    from nemo_amd.workloads import twelve_class_workload
    wl = twelve_class_workload(6, seed=9, cfg=SolverConfig(image_size=(256, 384), total_epochs=20), categories=['car', 'sofa'])
    s, eng = wl.solver, wl.solver.engine
    maps = eng.quantize(wl.feats)
    back = eng.dequantize(*maps)
    clutter = torch.nn.functional.normalize(torch.randn(5, 128, generator=torch.Generator().manual_seed(2))).cuda()
    a, b = s.solve_all(maps, clutter, wl.mesh_idx, clutter8=False), s.solve_all(back, clutter, wl.mesh_idx)
    assert torch.equal(a.campos, b.campos) and torch.equal(a.theta, b.theta) and torch.equal(a.loss, b.loss) and torch.equal(a.init_index, b.init_index)
    rounded = s.solve_all(maps, clutter, wl.mesh_idx)
    assert not torch.equal(a.loss, rounded.loss)
    want, bound = scores64(maps, clutter)
    assert bool(((eng.clutter_score(back, clutter).cpu().double() - want).abs() <= bound).all())
    off = (eng.q8_clutter_score(maps, eng.quantize(clutter)).cpu().double() - want).abs()
    assert bool((off > bound).any())                                          # the rounding is far outside it


def test_runner_keeps_the_clutter_vectors_of_a_record_in_8_bits(tmp_path):
    """The command on an 8-bit record, as on an f32 record of the same numbers, bit for bit; with --clutter8 it rounds the vectors too."""
    rng = np.random.default_rng(8)
    names, feats, mem, clu = {}, {}, {}, {}
    mesh_dir = tmp_path / 'mesh'
    mesh_dir.mkdir()
    for k, st in enumerate(('mesh01', 'mesh02')):
        v, f = syn.class_mesh('car', 300 + 50 * k)
        mesh_utils.save_off(str(mesh_dir / ('%02d.off' % (k + 1))), v, f)
        mem[st], clu[st] = syn.unit_rows(rng, len(v), 128), syn.unit_rows(rng, 6 + k, 128)
        names[st] = ['%s_%d' % (st, i) for i in range(7)]
        for n in names[st]:
            feats[n] = syn.unit_rows(rng, 12 * 23, 128).reshape(12, 23, 128).transpose(2, 0, 1).copy()
    src, in8, same = (str(tmp_path / n) for n in ('f32.npz', 'q8.npz', 'same.npz'))
    records.write_feature_record(src, mem, clu, names, feats)
    records.quantize_record(src, in8)
    with records.FeatureRecord(in8) as rec:
        records.write_feature_record(same, mem, clu, names, {n: rec.feature(n) for n in feats})

    def solve(record, *more):
        args = solve_all.build_parser().parse_args(['--type_', 'car', '--record_file', record, '--mesh_path', str(mesh_dir), '--image_size', '96,184',
                                                    '--total_epochs', '15', '--batch', '8', *more])
        got = solve_all.solve_category(args, 'cuda:0')
        return got[0], got[2], args
    want_names, want, _ = solve(same)
    got_names, got, args = solve(in8)
    assert got_names == want_names and np.array_equal(got, want)
    _, rounded, _ = solve(in8, '--clutter8')
    assert not np.array_equal(rounded, want)
    with records.FeatureRecord(in8) as rec:
        jobs = solve_all.category_jobs(rec, ['mesh01', 'mesh02'])
        a, _ = solve_all.solve_shard(args, rec, ['mesh01', 'mesh02'], *jobs, 'cuda:0', clutter8=True)
        b, info = solve_all.solve_shard(args, rec, ['mesh01', 'mesh02'], *jobs, 'cuda:0', clutter8=False)
        assert np.array_equal(a.cpu().numpy(), rounded) and np.array_equal(b.cpu().numpy(), want)
        for i, n in enumerate(jobs[0]):
            m = torch.from_numpy(clu['mesh%02d' % (jobs[1][i] + 1)]).mean(0)
            vec = (m / m.square().sum().sqrt())[None]
            score, bound = scores64(rec.feature8(n), vec)
            # the vector itself is computed in fp32 by the solver: 8 steps of it (mean, square, sum, root, quotient)
            off = (info['clu'][i].cpu().double() - score).abs()
            assert bool((off <= bound + 8 * 2.0 ** -23 * bound / (129 * 2.0 ** -23)).all())


def test_solver_refuses_clutter_vectors_of_another_length():
    """As with f32 maps: [K, D] or [D], and nothing that could be folded into that."""
    from nemo_amd.pose_solver import SolverConfig
    from nemo_amd.workloads import twelve_class_workload
    wl = twelve_class_workload(2, seed=9, cfg=SolverConfig(image_size=(256, 384), total_epochs=5), categories=['car'])
    s, eng = wl.solver, wl.solver.engine
    maps = eng.quantize(wl.feats)
    for shape in ((2, 256), (1, 2, 128), (256,), (256, 64)):
        for feats, c8 in ((maps, True), (maps, False), (wl.feats, True)):
            with pytest.raises(ValueError):
                s.solve_all(feats, torch.ones(shape, device='cuda'), wl.mesh_idx, clutter8=c8)
    vec = torch.nn.functional.normalize(torch.ones(1, 128)).cuda()
    for c8 in (True, False):
        a, b = s.solve_all(maps, vec, wl.mesh_idx, clutter8=c8), s.solve_all(maps, vec[0], wl.mesh_idx, clutter8=c8)
        assert torch.equal(a.campos, b.campos) and torch.equal(a.loss, b.loss)

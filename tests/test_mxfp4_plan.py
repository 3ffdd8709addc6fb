"""The sizes of test_gpu_mxfp4_sizes.py reach every form of the kernels that large weights run on (caifx_rows_plan.hpp, caifx_wide_plan.hpp)."""
import itertools

from test_gpu_mxfp4_sizes import DENSE, FEW

MX, DENSE_WEIGHT, BOTH = 0, 1, 2


def test_rows(mxfp4_plans):
    def forms(kind, weights, pieces, direct):
        return set(mxfp4_plans([(0, M, N, K, kind, weights, pieces, direct) for M, N, K in FEW]))
    for kind, direct in ((MX, 1), (MX, 0), (BOTH, 1)):
        got = forms(kind, 1, 1, direct)
        assert {f[:2] for f in got} >= {(16, 2), (16, 4), (32, 2), (32, 4), (64, 4)} and max(f[2] for f in got) > 1
    # fp32 in three pieces: 32 rows take two column tiles at most
    for direct in (0, 1):
        got = forms(MX, 1, 3, direct)
        assert {f[:2] for f in got} >= {(16, 2), (16, 4), (32, 2)}
    for kind, pieces in ((MX, 1), (MX, 3), (DENSE_WEIGHT, 1)):
        got = {f[:2] for f in forms(kind, 2, pieces, 1)}
        assert got >= ({(16, 2), (16, 4), (32, 2)} if pieces == 3 else {(16, 4), (32, 4), (64, 4)})


def up(v):
    return -(-v // 64) * 64


def test_dense(mxfp4_plans):
    gated = mxfp4_plans([(1, M, N, pieces * up(K), 1) for (M, N, K), pieces in itertools.product(DENSE, (1, 3))])
    assert {f[:2] for f in gated} == {(256, 256), (128, 256), (128, 128)}
    plain = mxfp4_plans([(1, M, N, up(K), 0) for M, N, K in DENSE + [(2048, 11001, 1088)]])
    assert {f[:2] for f in plain} == {(256, 256), (128, 256), (128, 128)}
    # both weights' gradient in one chain, whose steps several workgroups share
    chained = mxfp4_plans([(1, M, K, 2 * pieces * up(N), 0) for (M, N, K), pieces in itertools.product(DENSE, (1, 3))])
    assert {f[:2] for f in chained} == {(256, 256), (128, 256), (128, 128)} and max(f[2] for f in chained) > 1

"""A synchronous call on a session runs after every job submitted before it,
also when the worker has not taken the job up yet."""
import numpy as np
import pytest

from gpu_helpers import require_gpu
from shear_amd import datagen
from shear_amd import subtree as S

pytestmark = pytest.mark.gpu

DIM = 32


def _task(orc, n, seed):
    codes, scales, norms = orc.quantize(datagen.gmm_numpy(n, DIM, 8, 0.3, seed))
    gids = np.random.default_rng(seed).permutation(1 << 20)[:n].astype(np.uint32)
    return codes, scales, norms, gids


def _points(out, gids):
    return gids[out.leaf_row_ids[: out.leaf_rows].cpu().numpy().view(np.uint32)]


@pytest.mark.parametrize("jobs", [1, 2])
def test_a_run_right_after_submissions_uses_the_last_ones_rows(orc, jobs):
    require_gpu()
    params = S.PiPNNSubtreeParams(leaf_knn=16, c_max=256, psamp_fraction=0.01, fanout_second=2, random_seed=11)
    tasks = [_task(orc, 1500, seed) for seed in (3, 4)][:jobs]
    reqs = [S.GpuSubtreePartitionRequest(point_ids=t[3], parent_points=4500) for t in tasks]
    for _ in range(8):  # a new session each time: its worker's thread starts with the first job
        sess = S.SubtreeSession(0)
        deferred = [sess.submit_owned_quantized_subtree_l2_compact_topk(q, *t, DIM, params)
                    for q, t in zip(reqs, tasks)]
        out = sess.run(reqs[-1], params)
        results = [d.finish() for d in deferred]
        assert out.leaf_count == results[-1].leaf_count
        want = np.concatenate([b.point_ids for b in results[-1].compact_batches])
        assert np.array_equal(_points(out, tasks[-1][3]), want)
        sess.close()

"""Chunk attention and the windowed decode at the edges of what their arguments allow."""
import pytest
import torch

from attend_ref import Cache, check
from test_gpu_attend import Step, ops_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float32), (256, torch.float16)])
@pytest.mark.parametrize("n_splits", [1, 2, 7])
def test_rows_before_the_first_sequence(D, dtype, n_splits):
    """query_start_loc[0] > 0: rows that belong to no sequence stay as they are, whether or not the keys are split."""
    ops = ops_of(D, 4, 4, dtype, 16)
    c = Cache(ops, [300, 40], 2, seed=5)
    step = Step(c, [3, 9, 140], seed=2, spare=2)                               # 3 rows of nobody, then the two sequences
    step.qsl, step.seq_lens = step.qsl[1:], torch.tensor([309, 180], dtype=torch.int32, device="cuda")
    rows = step.q.shape[0]
    out = torch.full((rows, 8, D), 7.0, dtype=dtype, device="cuda")
    work = torch.full((ops.chunk_work_size(rows, 2, n_splits),), float("nan"), device="cuda")
    ops.attend_chunk(step.q, step.k, step.v, out, step.qsl, step.seq_lens, c.tail_idx, c.pool, c.block_table, c.tail_k, D ** -0.5,
                     n_splits, work)
    torch.cuda.synchronize()
    assert (out[:3] == 7.0).all() and (out[152:] == 7.0).all()
    own = Step(c, [9, 140], seed=2, spare=0)
    own.q, own.k, own.v = (t[3:152] for t in (step.q, step.k, step.v))
    check(out[3:152], *own.reference(None, 0), dtype, f"rows 3.. splits {n_splits}")

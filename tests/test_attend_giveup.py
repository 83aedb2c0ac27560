"""Chunk attention whose waits run out: NaN for what a block did not finish, the error flag, and a context that goes on."""
import ctypes

import pytest
import torch

P16 = ctypes.c_void_p(16)


@pytest.mark.parametrize("kw", [dict(slot=2), dict(slot=-1), dict(tile=-1), dict(limit=0), dict(limit=2001), dict(D=64), dict(bits=8), dict(page=32),
                                dict(dtype=0), dict(q=None)])
def test_refusals(kw):
    from kushkash_b200._cuda import KUSH_ERR_ARG, KUSH_ERR_UNSUPPORTED, last_error, lib
    a = dict(D=128, bits=4, page=16, dtype=1, group=4, q=P16, qs=512, k=P16, v=P16, ks=128, vs=128, out=P16, qsl=P16, seq_lens=P16,
             tail_idx=P16, cache=P16, bs=2624, hs=2624, tail_k=P16, table=P16, max_pages=4, hkv=1, scale=0.1, window=0, sinks=0,
             n_splits=1, ml=None, o=None, rows=4, seqs=1, slot=0, tile=0, limit=50)
    a.update(kw)
    rc = lib().kush_sm100_attend_chunk_held(*a.values(), None)
    assert rc in (KUSH_ERR_ARG, KUSH_ERR_UNSUPPORTED) and last_error()


# (history, new rows, group): up to 128 rows both slots hold the same rows and take the key tiles in turn, above each its own.
# 8 tiles: slot 0 has finished its last when slot 1's is kept back.
@pytest.mark.gpu
@pytest.mark.parametrize("ctx,new,G,slot,tile", [(1000, 5, 4, 1, 3), (1000, 5, 4, 0, 3), (1000, 5, 4, 1, 0), (1000, 1, 1, 0, 0), (40, 200, 1, 1, 0),
                                                 (40, 200, 1, 0, 1), (700, 64, 4, 1, 2)])
def test_a_wait_that_runs_out(ctx, new, G, slot, tile):
    from attend_ref import Cache
    from kushkash_b200 import _cuda
    from test_gpu_attend import Step, ops_of
    ops = ops_of(128, 4, G, torch.bfloat16, 16)
    c = Cache(ops, [ctx], 2, seed=4)
    step = Step(c, [new], seed=1, spare=3)
    want = step.run()
    assert _cuda.device_error() == 0
    run = ops._run
    ops._run = lambda entry, *args: run(entry + "_held", *args, slot, tile, 30)
    got = step.run()                                                           # (rows behind the last sequence are checked there)
    ops._run = run
    assert _cuda.device_error() == 8
    nan, rows = got.isnan().all(-1), torch.arange(new * G).view(new, G).repeat(1, 2).cuda()
    assert torch.equal(got[~nan], want[~nan])                                  # finished before, or not written at all
    assert nan.all() if new * G <= 128 else nan[(rows >= 128) == (slot == 1)].all()
    assert torch.equal(step.run(), want) and _cuda.device_error() == 0         # the context and the next launch are as before


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.1, 60.0])
def test_a_part_that_gave_up_is_not_dropped(scale):
    """11 key tiles in two parts of 6 and 5: only the first has a third tile for slot 1.  The merged rows are NaN, however large
    the other part's scores are."""
    from attend_ref import Cache
    from kushkash_b200 import _cuda
    from test_gpu_attend import Step, ops_of
    ops = ops_of(128, 4, 4, torch.bfloat16, 16)
    c = Cache(ops, [1380], 2, seed=4)
    step = Step(c, [10], seed=1, spare=0)
    out = torch.zeros(10, 8, 128, dtype=torch.bfloat16, device="cuda")
    work = torch.zeros(ops.chunk_work_size(10, 2, 2), device="cuda")
    args = (step.q, step.k, step.v, out, step.qsl, step.seq_lens, c.tail_idx, c.pool, c.block_table, c.tail_k, scale, 2, work)
    ops.attend_chunk(*args)
    torch.cuda.synchronize()
    assert not out.isnan().any() and _cuda.device_error() == 0
    if scale > 1:
        m = work[10 * 2 * 2 * 4 * 128:].view(10, 2, 2, 4, 2)[..., 0]           # the parts' maxima, in nats
        assert (m[:, :, 1] > 110).any()
    run = ops._run
    ops._run = lambda entry, *a: run(entry + "_held", *a, 1, 2, 30)
    ops.attend_chunk(*args)
    torch.cuda.synchronize()
    assert out.isnan().all() and _cuda.device_error() == 8

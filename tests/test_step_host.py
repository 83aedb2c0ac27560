"""What rope and attend_chunk refuse before anything is launched, on CPU tensors: an Ops object whose launches are recorded."""
import pytest
import torch

D, G, H, P, S, ROWS = 64, 2, 3, 16, 2, 5


@pytest.fixture
def ops():
    from kushkash_b200 import GpuConfig, Ops
    o = Ops.__new__(Ops)
    o.device, o.dev = torch.device("cpu"), torch.zeros(1).get_device()
    o.D, o.bits, o.G, o.dtype, o.P, o._fmt = D, 4, G, torch.float16, P, (D, 4, P, 0)
    o.cfg = GpuConfig(D, 4, G, "float16", "sm_100a", P)
    o.calls = []
    o._run = lambda entry, *args: o.calls.append((entry, args))
    return o


def test_rope_outputs(ops):
    plan, pos = ops.rotary(), torch.arange(ROWS)
    x = torch.zeros(ROWS, H, D, dtype=torch.float16)
    wide = torch.zeros(ROWS, 2 * H * D, dtype=torch.float16)
    flat = torch.zeros(ROWS * H * D, dtype=torch.float16)
    for q, q_out in ((x, None), (x, x), (x, torch.empty_like(x)), (wide[:, :H * D].view(ROWS, H, D), wide[:, H * D:].view(ROWS, H, D)),
                     (wide[:, :H * D].view(ROWS, H, D), wide[:, :H * D].view(ROWS, H, D)),
                     (x[:1].expand(ROWS, H, D), torch.empty_like(x))):
        ops.rope(q, None, pos, plan, q_out)
        assert ops.calls.pop()[0] == "kush_sm100_rope"
    ops.rope(x[:1], None, pos[:1], plan, wide[:1, :H * D].view(1, H, D))
    ops.rope(x[:1], None, pos[:1], plan, flat.view(ROWS, H, D)[:1])
    ops.calls.clear()
    for q, q_out in ((x, torch.zeros(1, H, D, dtype=torch.float16).expand(ROWS, H, D)),       # every row into one
                     (x, torch.zeros(ROWS, 1, D, dtype=torch.float16).expand(ROWS, H, D)),
                     (x[:1].expand(ROWS, H, D), x),                                           # the first row is read while it is written
                     (flat.view(ROWS, H, D), flat.view(H, ROWS, D).transpose(0, 1))):         # the same memory in another order
        with pytest.raises(ValueError, match="rope"):
            ops.rope(q, None, pos, plan, q_out)
        with pytest.raises(ValueError, match="rope"):
            ops.rope(None, q, pos, plan, None, q_out)
    assert not ops.calls


def arguments(**kw):
    i32 = torch.int32
    a = dict(q=torch.zeros(ROWS, H * G, D, dtype=torch.float16), k=torch.zeros(ROWS, H, D, dtype=torch.float16),
             v=torch.zeros(ROWS, H, D, dtype=torch.float16), out=torch.zeros(ROWS, H * G, D, dtype=torch.float16),
             query_start_loc=torch.tensor([0, 2, 5], dtype=i32), seq_lens=torch.ones(S, dtype=i32), tail_idx=torch.zeros(S, dtype=i32),
             cache=torch.zeros(5, H, P * D + 4 * D + 4 * P, dtype=torch.uint8), block_table=torch.zeros(S, 2, dtype=i32),
             tail_k=torch.zeros(S, H, P, D, dtype=torch.float16), scale=0.125)
    a.update(kw)
    return a


def test_chunk_arguments(ops):
    ops.attend_chunk(**arguments())
    ops.attend_chunk(**arguments(cache=torch.zeros(5, H + 1, 1344, dtype=torch.uint8)))
    assert len(ops.calls) == 2
    for kw in (dict(cache=torch.zeros(5, H - 1, 1344, dtype=torch.uint8)), dict(cache=torch.zeros(5000, dtype=torch.uint8)),
               dict(tail_idx=torch.zeros((), dtype=torch.int32)), dict(block_table=torch.zeros(2 * S, dtype=torch.int32)),
               dict(seq_lens=torch.ones(S, 1, dtype=torch.int32))):
        with pytest.raises(ValueError, match="attend_chunk"):
            ops.attend_chunk(**arguments(**kw))
    assert len(ops.calls) == 2


@pytest.mark.parametrize("dim,dtype,seqs,rows,longest,window,want", [
    (128, torch.bfloat16, 1, 17, 517, None, 2), (64, torch.float16, 16, 80, 4005, None, 1),        # tensor cores: chunk_split_factor
    (128, torch.float32, 1, 17, 517, None, 10), (256, torch.bfloat16, 1, 17, 517, None, 10),       # 24 blocks of 32 rows
    (128, torch.float32, 1, 1, 8001, None, 74), (256, torch.bfloat16, 1, 1, 8001, 1000, 20),       # filled once; the window's tokens
    (64, torch.float32, 16, 80, 4005, None, 8), (128, torch.float32, 16, 80, 4005, None, 15),
    (256, torch.float16, 16, 80, 4005, None, 9), (256, torch.bfloat16, 5, 500, 300, None, 1), (128, torch.float32, 1, 2048, 9000, None, 1),
    (64, torch.float32, 0, 0, 0, None, 1)])
def test_chunk_splits_follow_the_kernels(dim, dtype, seqs, rows, longest, window, want):
    from kushkash_b200 import Ops
    o = Ops.__new__(Ops)
    o.D, o.G, o.dtype, o.sms = dim, 4, dtype, 148
    assert o.chunk_splits(rows, seqs, 8, longest, window=window) == want

"""What the windowed decode refuses before anything is launched, on CPU tensors: an Ops object whose launches are recorded."""
import pytest
import torch

D, G, H, P, S = 64, 2, 3, 16, 4


@pytest.fixture
def ops():
    from kushkash_b200 import Ops
    o = Ops.__new__(Ops)
    o.device = torch.device("cpu")
    o.D, o.bits, o.G, o.dtype, o.P, o._fmt = D, 4, G, torch.float16, P, (D, 4, P, 0)
    o.calls = []
    o._run = lambda entry, *args: o.calls.append((entry, args))

    def here(what, *tensors):                                                  # (other devices than the CPU: "meta")
        if any(t.device != o.device for t in tensors):
            raise ValueError(f"{what}: every tensor must be on {o.device}")

    o._here = here
    return o


def arguments(**kw):
    i32 = torch.int32
    rb = P * D + 4 * D + 4 * P
    a = dict(q=torch.zeros(S, H * G, D, dtype=torch.float16), out=torch.zeros(S, H * G, D, dtype=torch.float16),
             cache=torch.zeros(5, H, rb, dtype=torch.uint8), block_table=torch.zeros(S, 2, dtype=i32),
             seq_lens=torch.ones(S, dtype=i32), tail_idx=torch.zeros(S, dtype=i32),
             tail_k=torch.zeros(S, H, P, D, dtype=torch.float16), scale=0.125, window=8, sinks=2)
    a.update(kw)
    return a


def test_good_calls_launch(ops):
    work = torch.zeros(ops.work_size(S, H, 2, fused=True))
    table = torch.zeros(S + 1, 7, dtype=torch.int32)[:, :5]                    # rows apart, more sequences than q has
    for kw in ({}, dict(n_splits=2, work=work), dict(n_splits=2, work=work, fused=True), dict(block_table=table),
               dict(order=torch.arange(S, dtype=torch.int32)), dict(seq_lens=torch.ones(S + 2, dtype=torch.int32)),
               dict(window=2 ** 40, sinks=2 ** 40)):
        ops.decode(**arguments(**kw))
        entry, args = ops.calls.pop()
        assert entry == "kush_sm100_decode_window" and not ops.calls
        assert args[5] and args[14] == kw.get("block_table", torch.zeros(S, 2)).stride(0) and args[21] == S


PACKED = torch.zeros(S, (G + 2) * H * D, dtype=torch.float16)


@pytest.mark.parametrize("kw", [
    dict(q=PACKED[:, :G * H * D].view(S, H * G, D)),                           # a part of q|k|v rows
    dict(out=PACKED[:, :G * H * D].view(S, H * G, D)), dict(q=torch.zeros(S, H * G, D)), dict(out=torch.zeros(S, H * G, D)),
    dict(q=torch.zeros(S, H * G, D, dtype=torch.bfloat16)), dict(q=torch.zeros(S, H * G + 1, D, dtype=torch.float16)),
    dict(q=torch.zeros(S, H * G * D, dtype=torch.float16)), dict(out=torch.zeros(S - 1, H * G, D, dtype=torch.float16)),
    dict(tail_k=torch.zeros(S, H, P, D)), dict(tail_k=torch.zeros(S, H, 32, D, dtype=torch.float16)),
    dict(tail_k=torch.zeros(S, P, H, D, dtype=torch.float16).transpose(1, 2)),
    dict(seq_lens=torch.ones(S, dtype=torch.int64)), dict(tail_idx=torch.zeros(S, dtype=torch.int64)),
    dict(block_table=torch.zeros(S, 2, dtype=torch.int64)), dict(seq_lens=torch.ones(S - 1, dtype=torch.int32)),
    dict(seq_lens=torch.ones(2 * S, dtype=torch.int32)[::2]), dict(tail_idx=torch.zeros(2 * S, dtype=torch.int32)[::2]),
    dict(tail_idx=torch.zeros(S - 1, dtype=torch.int32)), dict(block_table=torch.zeros(S - 1, 2, dtype=torch.int32)),
    dict(block_table=torch.zeros(2, S, dtype=torch.int32).T), dict(block_table=torch.zeros(2 * S, dtype=torch.int32)),
    dict(cache=torch.zeros(5, H - 1, 1344, dtype=torch.uint8)),
    dict(n_splits=2), dict(n_splits=2, work=torch.zeros(10)), dict(n_splits=2, work=torch.zeros(10000, dtype=torch.float16)),
    dict(n_splits=2, work=torch.zeros(10000, device="meta")), dict(order=torch.arange(S, dtype=torch.int32, device="meta")),
    dict(order=torch.arange(S)), dict(order=torch.arange(S + 1, dtype=torch.int32)), dict(window=None), dict(window=0),
    dict(sinks=-1)])
def test_refusals(ops, kw):
    with pytest.raises(ValueError, match="decode"):
        ops.decode(**arguments(**kw))
    assert not ops.calls


def test_refused_work_of_a_fused_merge(ops):
    with pytest.raises(ValueError, match="decode"):                            # no room for the counters
        ops.decode(**arguments(n_splits=2, fused=True, work=torch.zeros(ops.work_size(S, H, 2))))
    assert not ops.calls


@pytest.mark.parametrize("D,bits,G,dtype,page,seqs,heads,window,want", [
    (128, 4, 4, torch.bfloat16, 16, 1, 8, 8192, 32), (128, 8, 7, torch.float16, 32, 61, 4, 1000, 1), (128, 8, 7, torch.float16, 32, 30, 4, 1000, 2),
    (64, 4, 16, torch.bfloat16, 16, 4, 8, 4096, 9), (64, 4, 16, torch.bfloat16, 16, 61, 4, 1000, 1),      # two CTAs an SM, though four fit
    (256, 8, 4, torch.bfloat16, 32, 4, 8, 4096, 4), (256, 8, 4, torch.bfloat16, 32, 30, 4, 1000, 1),      # one CTA an SM
    (256, 4, 4, torch.bfloat16, 16, 4, 8, 4096, 9),
    (128, 4, 4, torch.float32, 16, 4, 8, 4096, 18), (128, 4, 4, torch.float32, 16, 1, 8, 8192, 51),       # the CUDA cores' own rule
    (128, 4, 40, torch.bfloat16, 32, 1, 8, 8192, 37), (64, 8, 4, torch.float32, 32, 61, 4, 1000, 4), (256, 4, 12, torch.bfloat16, 16, 61, 4, 1000, 1),
    (256, 4, 1, torch.float32, 16, 1, 1, 100, 1), (64, 4, 1, torch.float32, 16, 0, 1, 100, 1)])
def test_splits_follow_the_kernels(D, bits, G, dtype, page, seqs, heads, window, want):
    from kushkash_b200 import GpuConfig, Ops
    o = Ops.__new__(Ops)
    o.D, o.bits, o.G, o.dtype, o.P, o.sms = D, bits, G, dtype, page, 148
    o.cfg = GpuConfig(D, bits, G, str(dtype)[6:], "sm_100a", page)
    assert o.splits(seqs, heads, 100000 // page, window=window) == want
    assert o.splits(seqs, heads, 0, window=window) == 1

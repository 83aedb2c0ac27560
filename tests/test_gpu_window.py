"""Decode under a sliding window with sink tokens, against the definition in 64 bits."""
import pytest
import torch

from attend_ref import Cache, attend, check

pytestmark = pytest.mark.gpu


def ops_of(D, bits, G, dtype, P):
    from kushkash_b200 import Ops
    return Ops(torch.device("cuda:0"), D, bits, G, dtype, P)


def unit(dtype, D, G):
    """(u, c_s) of attend(): the tensor-core kernel rounds q and k to fp16 (two roundings of the score's terms and the
    subtraction of the reference bias: 4), the fp32 kernel adds D terms."""
    return (2.0 ** -24, D + 16.0) if dtype == torch.float32 else (2.0 ** -11, 4.0)


def reference(c, q, window, sinks, u, c_s):
    H, G, D = c.H, c.ops.G, c.ops.D
    out, bound = torch.zeros(len(c.lens), H * G, D, dtype=torch.float64), torch.zeros(len(c.lens), H * G, D, dtype=torch.float64)
    for s, n in enumerate(c.lens):
        if n == 0:
            continue
        k, v = c.tokens(s)
        lo = max(0, n - window)
        ref = c.kb_all[c.table_cpu[s, :n // c.ops.P].long()].abs().amax(0) if n >= c.ops.P else None
        see = torch.tensor([j for j in range(n) if j >= lo or j < sinks])
        o, b = attend(q[s].cpu().view(1, H, G, D), k[see], v[see], torch.tensor([n - 1]), see, D ** -0.5, window, sinks, ref, u,
                      c_s)
        out[s], bound[s] = o.view(H * G, D), b.view(H * G, D)
    return out, bound


def run(c, q, window, sinks, n_splits=1, fused=False, **kw):
    ops, S, H = c.ops, len(c.lens), c.H
    out = torch.full_like(q, float("nan"))
    work = torch.zeros(ops.work_size(S, H, n_splits, fused=True), dtype=torch.float32, device=q.device) if n_splits > 1 else None
    if work is not None:
        work[:ops.work_size(S, H, n_splits)] = float("nan")
    ops.decode(q, out, c.pool, c.block_table, c.seq_lens, c.tail_idx, c.tail_k, ops.D ** -0.5, n_splits, work, window=window,
               sinks=sinks, fused=fused, **kw)
    torch.cuda.synchronize()
    return out


LENS = [0, 1, 15, 16, 17, 31, 32, 33, 64, 100, 257, 700]


@pytest.mark.parametrize("D,bits,G,dtype,P", [
    (128, 4, 4, torch.bfloat16, 16), (128, 4, 4, torch.bfloat16, 32), (128, 8, 7, torch.float16, 32), (64, 4, 1, torch.float16, 16),
    (64, 8, 12, torch.bfloat16, 16), (256, 4, 2, torch.bfloat16, 32), (256, 8, 8, torch.float16, 16),
    (128, 4, 4, torch.float32, 16), (64, 8, 3, torch.float32, 32), (128, 4, 40, torch.bfloat16, 32), (256, 8, 5, torch.float32, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 16), (33, 40), (100, 4), (256, 64), (5000, 7), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_window_decode(D, bits, G, dtype, P, window, sinks):
    ops = ops_of(D, bits, G, dtype, P)
    c = Cache(ops, LENS, 2, seed=D + bits + P, strided=P == 32)
    c.hide([n - 1 for n in c.lens], window, sinks)
    q = torch.randn(len(LENS), 2 * G, D, generator=torch.Generator().manual_seed(7)).to(dtype).cuda()
    want, bound = reference(c, q, window, sinks, *unit(dtype, D, G))
    for n_splits, fused in ((1, False), (3, False), (4, True), (30, False)):
        got = run(c, q, window, sinks, n_splits, fused)
        check(got, want, bound, dtype, f"window {window} sinks {sinks} splits {n_splits}{' fused' if fused else ''}")
        assert (got[0] == 0).all()                                             # the empty sequence


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_window_covering_everything_is_the_plain_decode(dtype):
    ops = ops_of(128, 4, 4, dtype, 16)
    c = Cache(ops, LENS, 3, seed=1)
    q = torch.randn(len(LENS), 12, 128, device="cuda", dtype=torch.float32).to(dtype)
    plain = torch.empty_like(q)
    ops.decode(q, plain, c.pool, c.block_table, c.seq_lens, c.tail_idx, c.tail_k, 128 ** -0.5)
    got = run(c, q, 700, 0)
    if dtype == torch.bfloat16:
        assert torch.equal(got, plain)                                         # the same tiles in the same order
    else:
        assert (got - plain).abs().max() < 1e-4                                # another kernel, both in fp32


@pytest.mark.parametrize("n_splits", [1, 4])
@pytest.mark.parametrize("dtype,G", [(torch.bfloat16, 4), (torch.float32, 2)])
def test_window_decode_rotated_and_ordered(n_splits, dtype, G):
    """rotate=True over a cache of rotated rows: the same as rotating q before and the output after."""
    ops = ops_of(128, 4, G, dtype, 16)
    c = Cache(ops, LENS, 2, seed=5)
    q = torch.randn(len(LENS), 2 * G, 128, device="cuda").to(dtype)
    order = ops.longest_first(c.seq_lens)
    got = run(c, q, 90, 6, n_splits, rotate=True, order=order)
    base = run(c, ops.fwht(q), 90, 6, n_splits)
    want = ops.fwht(base).double().cpu()
    # fwht(q) rounds q to the type once more and the two outputs round twice more; the transform keeps norms
    u = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2.0 ** -20
    k_mass = 40.0                                                              # |q| |k| scale of these scores, at most
    assert (got.double().cpu() - want).norm() <= (3 + 2 * k_mass) * u * want.norm() + 1e-6
    assert torch.equal(run(c, q, 90, 6, n_splits, order=order), run(c, q, 90, 6, n_splits))


def test_window_in_a_graph_and_on_a_stream():
    ops = ops_of(128, 8, 4, torch.bfloat16, 32)
    c = Cache(ops, [300, 77, 1200], 2, seed=3)
    q = torch.randn(3, 8, 128, device="cuda").to(torch.bfloat16)
    want = run(c, q, 200, 5, 4)
    work = torch.empty(ops.work_size(3, 2, 4), dtype=torch.float32, device="cuda")
    out, side = torch.zeros_like(q), torch.cuda.Stream()
    args = (c.pool, c.block_table, c.seq_lens, c.tail_idx, c.tail_k, 128 ** -0.5, 4, work)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.decode(q, out, *args, window=200, sinks=5)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.decode(q, out, *args, window=200, sinks=5)
    q.copy_(torch.randn_like(q))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, run(c, q, 200, 5, 4))


def test_window_refusals():
    ops = ops_of(128, 4, 4, torch.bfloat16, 16)
    c = Cache(ops, [40], 1, seed=2)
    q = torch.randn(1, 4, 128, device="cuda").to(torch.bfloat16)
    for kw in (dict(window=0), dict(window=-3), dict(window=None, sinks=2), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            ops.decode(q, torch.empty_like(q), c.pool, c.block_table, c.seq_lens, c.tail_idx, c.tail_k, 0.1, **kw)
    with pytest.raises(ValueError):
        ops.decode(q, torch.empty_like(q), c.pool, c.block_table, c.seq_lens, c.tail_idx, c.tail_k, 0.1, 2, None, window=4)
    with pytest.raises(ValueError):
        ops.decode(q, torch.empty_like(q), c.pool, c.block_table, c.seq_lens.cpu(), c.tail_idx, c.tail_k, 0.1, window=4)

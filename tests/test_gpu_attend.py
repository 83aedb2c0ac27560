"""Chunk attention over the packed cache and the new rows, against the definition in 64 bits."""
import pytest
import torch

from attend_ref import Cache, attend, check

pytestmark = pytest.mark.gpu


def ops_of(D, bits, G, dtype, P):
    from kushkash_b200 import Ops
    return Ops(torch.device("cuda:0"), D, bits, G, dtype, P)


def unit(dtype, D):
    """(u, c_s) of attend(): the tensor-core kernel rounds keys (after the subtraction of the reference bias) to fp16 and
    takes q as it is: two roundings of what enters a score; the fp32 kernel adds D terms."""
    return (2.0 ** -24, D + 16.0) if dtype == torch.float32 else (2.0 ** -11, 3.0)


class Step:
    """New rows of a step over a cache, inside wider rows, with NaN rows behind the last sequence."""

    def __init__(self, c, new, seed, spare=5):
        ops, H = c.ops, c.H
        g = torch.Generator().manual_seed(seed)
        self.c, self.new = c, list(new)
        rows, D = sum(new) + spare, ops.D
        qkv = torch.full((rows, (ops.G + 2) * H * D + 16), float("nan"), dtype=ops.dtype)
        qkv[:sum(new)] = torch.randn(sum(new), qkv.shape[1], generator=g).to(ops.dtype)
        qkv[:sum(new), ops.G * H * D:(ops.G + 1) * H * D] += 2 * torch.randn(H * D, generator=g).to(ops.dtype)
        qkv = qkv.cuda()
        self.q, self.k, self.v = (qkv[:, a * H * D:b * H * D].view(rows, -1, D)
                                  for a, b in ((0, ops.G), (ops.G, ops.G + 1), (ops.G + 1, ops.G + 2)))
        self.qsl = torch.tensor([0] + self.new).cumsum(0).to(torch.int32).cuda()
        self.seq_lens = torch.tensor([a + b for a, b in zip(c.lens, self.new)], dtype=torch.int32).cuda()

    def run(self, window=None, sinks=0, n_splits=1):
        c, ops = self.c, self.c.ops
        rows = self.q.shape[0]
        out = torch.full((rows, c.H * ops.G, ops.D), 7.0, dtype=ops.dtype, device="cuda")
        work = None
        if n_splits > 1:
            work = torch.full((ops.chunk_work_size(rows, c.H, n_splits),), float("nan"), device="cuda")
        ops.attend_chunk(self.q, self.k, self.v, out, self.qsl, self.seq_lens, c.tail_idx, c.pool, c.block_table, c.tail_k,
                         ops.D ** -0.5, n_splits, work, window=window, sinks=sinks)
        torch.cuda.synchronize()
        assert (out[sum(self.new):] == 7.0).all(), "rows behind the last sequence were written"
        return out[:sum(self.new)]

    def reference(self, window, sinks):
        c, ops = self.c, self.c.ops
        H, G, D = c.H, ops.G, ops.D
        u, c_s = unit(ops.dtype, D)
        outs, bounds, row = [], [], 0
        for s, (n, t) in enumerate(zip(c.lens, self.new)):
            k, v = c.tokens(s)
            pos_q, pos_k = n + torch.arange(t), torch.arange(n + t)
            see = torch.ones(n + t, dtype=torch.bool)
            if window is not None:
                see = (pos_k > n - window) | (pos_k < sinks)
            kn, vn = self.k[row:row + t].cpu().double(), self.v[row:row + t].cpu().double()
            ref = c.kb_all[c.table_cpu[s, :n // ops.P].long()].abs().amax(0) if n >= ops.P else None
            if t:
                o, b = attend(self.q[row:row + t].cpu().view(t, H, G, D), torch.cat([k, kn])[see], torch.cat([v, vn])[see],
                              pos_q, pos_k[see], D ** -0.5, window, sinks, ref, u, c_s)
                outs.append(o.reshape(t, H * G, D))
                bounds.append(b.reshape(t, H * G, D))
            row += t
        return torch.cat(outs), torch.cat(bounds)


FORMS = [(128, 4, 4, torch.bfloat16, 16), (128, 4, 4, torch.bfloat16, 32), (128, 8, 7, torch.float16, 16), (128, 8, 1, torch.bfloat16, 32),
         (64, 4, 5, torch.float16, 32), (64, 8, 16, torch.bfloat16, 16), (256, 4, 2, torch.bfloat16, 16),
         (128, 4, 3, torch.float32, 16), (64, 8, 4, torch.float32, 32), (256, 8, 1, torch.float32, 32), (128, 4, 40, torch.bfloat16, 32),
         (64, 4, 150, torch.float16, 16)]
CTX = [0, 0, 1, 15, 16, 31, 33, 128, 130, 300, 513]
NEW = [1, 37, 3, 1, 130, 0, 17, 2, 64, 5, 129]


@pytest.mark.parametrize("D,bits,G,dtype,P", FORMS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (20, 3), (64, 70), (200, 16)])
def test_chunk(D, bits, G, dtype, P, window, sinks):
    ops = ops_of(D, bits, G, dtype, P)
    c = Cache(ops, CTX, 2, seed=D + bits, strided=P == 16)
    if window is not None:
        c.hide(c.lens, window, sinks)
    step = Step(c, NEW, seed=G)
    want, bound = step.reference(window, sinks)
    for n_splits in (1, 2, 5):
        check(step.run(window, sinks, n_splits), want, bound, dtype, f"chunk window {window} sinks {sinks} splits {n_splits}")


@pytest.mark.parametrize("ctx,new", [(0, 1), (0, 127), (0, 128), (0, 129), (127, 1), (128, 1), (129, 127), (1000, 1), (1023, 700),
                                     (2050, 33)])
@pytest.mark.parametrize("dtype,G", [(torch.bfloat16, 4), (torch.float16, 7)])
def test_chunk_lengths(ctx, new, dtype, G):
    """One sequence at every border of row tiles, key tiles and pages."""
    ops = ops_of(128, 4, G, dtype, 32)
    c = Cache(ops, [ctx], 1, seed=ctx)
    step = Step(c, [new], seed=new)
    want, bound = step.reference(None, 0)
    for n_splits in (1, 3):
        check(step.run(None, 0, n_splits), want, bound, dtype, f"chunk {ctx} + {new} splits {n_splits}")


def test_chunk_then_write_then_decode():
    """A serving step as it is used: rope, chunk attention, write; then one token: rope, append, windowed decode."""
    D, G, H, P, dt = 128, 4, 2, 16, torch.bfloat16
    ops = ops_of(D, 4, G, dt, P)
    c = Cache(ops, [45, 0, 200], H, seed=4, pad_blocks=40)
    new = [20, 33, 1]
    pages = [-(-(a + b + 1) // P) for a, b in zip(c.lens, new)]
    table, spare = c.table_cpu.clone(), iter(sorted(set(range(1, c.pool.shape[0])) - set(c.table_cpu.flatten().tolist())))
    table = torch.nn.functional.pad(table, (0, 8))
    for s, n in enumerate(pages):
        for p in range(-(-c.lens[s] // P), n):
            table[s, p] = next(spare)
    c.block_table = table.cuda()
    c.table_cpu = table
    step = Step(c, new, seed=9, spare=0)
    plan = ops.rotary(scaling={"rope_type": "linear", "factor": 2.0})
    pos = torch.cat([n + torch.arange(t) for n, t in zip(c.lens, new)]).cuda()
    step.q, step.k = ops.rope(step.q, step.k, pos, plan)
    want, bound = step.reference(50, 4)
    check(step.run(50, 4), want, bound, dt, "step chunk")
    js, jp, _ = ops.write_jobs(step.qsl, step.seq_lens, sum(new) // P + 6)
    ops.write(step.k, step.v, step.qsl, step.seq_lens, c.tail_idx, js, jp, c.pool, c.block_table, c.tail_k)
    q1, k1, v1 = (torch.randn(3, h, D, device="cuda").to(dt) for h in (H * G, H, H))
    q1, k1 = ops.rope(q1, k1, step.seq_lens, plan)
    ops.append(k1, v1, step.seq_lens, c.tail_idx, c.pool, c.block_table, c.tail_k, 0, True)
    out = torch.empty_like(q1)
    ops.decode(q1, out, c.pool, c.block_table, step.seq_lens, c.tail_idx, c.tail_k, D ** -0.5, window=50, sinks=4)
    torch.cuda.synchronize()
    from attend_ref import dequantize
    c.lens = step.seq_lens.tolist()
    assert c.lens == [66, 34, 202]
    c.k_all, c.v_all, c.kb_all = dequantize(c.pool, D, 4, P)
    c.tail_cpu = c.tail_k.cpu()
    for s, n in enumerate(c.lens):
        k, v = c.tokens(s)
        o, b = attend(q1[s:s + 1].cpu().view(1, H, G, D), k, v, torch.tensor([n - 1]), torch.arange(n), D ** -0.5, 50, 4,
                      c.kb_all[c.table_cpu[s, :n // P].long()].abs().amax(0), 2.0 ** -11, 4.0)
        check(out[s:s + 1], o.view(1, H * G, D), b.view(1, H * G, D), dt, f"step decode {s}")


def test_chunk_agrees_with_unpack():
    """The same keys and values as unpack() gives, attended with torch in fp32."""
    D, G, H, P, dt = 64, 4, 2, 32, torch.float16
    ops = ops_of(D, 8, G, dt, P)
    c = Cache(ops, [70, 5], H, seed=6)
    step = Step(c, [9, 40], seed=3, spare=0)
    got = step.run()
    plan = ops.unpack_plan(step.qsl, step.seq_lens, c.tail_idx, c.block_table, 4, 2, 49)
    kp, vp = (torch.zeros(124, H, D, dtype=dt, device="cuda") for _ in range(2))
    ops.unpack(c.pool, plan["page_blk"], plan["page_dst"], plan["tail_blk"], plan["tail_info"], c.tail_k,
               step.k.contiguous(), step.v.contiguous(), plan["new_dst"], kp, vp, False)
    row = 0
    for s, t in enumerate(step.new):
        a, b = plan["kv_start"][s:s + 2].tolist()
        n = c.lens[s]
        q = step.q[row:row + t].float().view(t, H, G, D)
        x = torch.einsum("thgd,nhd->thgn", q, kp[a:b].float()) * D ** -0.5
        x = x.masked_fill((torch.arange(n + t)[None] > n + torch.arange(t)[:, None]).cuda()[:, None, None], -torch.inf).softmax(-1)
        want = torch.einsum("thgn,nhd->thgd", x, vp[a:b].float()).reshape(t, H * G, D)
        assert (got[row:row + t].float() - want).norm() <= 4 * 2.0 ** -11 * 4 * want.norm()
        row += t


def test_chunk_graph_and_stream():
    ops = ops_of(128, 4, 4, torch.bfloat16, 16)
    c = Cache(ops, [100, 333], 2, seed=8)
    step = Step(c, [40, 7], seed=1, spare=2)
    rows, out = 49, torch.full((49, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    work = torch.empty(ops.chunk_work_size(rows, 2, 3), device="cuda")

    def call():
        ops.attend_chunk(step.q, step.k, step.v, out, step.qsl, step.seq_lens, c.tail_idx, c.pool, c.block_table, c.tail_k,
                         128 ** -0.5, 3, work)

    want = step.run(n_splits=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    assert torch.equal(out[:47], want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    step.q[:47] = torch.randn_like(step.q[:47])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[:47], step.run(n_splits=3)) and (out[47:] == 7.0).all()


@pytest.mark.parametrize("order", ["rising", "falling", "both"])
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("ctx", [0, 260])
def test_chunk_scores_that_move_the_maximum(order, D, dtype, ctx):
    """Scores that rise by about one per token, so that every 32 columns pass the running maximum by more than its slack,
    fall, or rise for some rows and fall for others."""
    ops = ops_of(D, 8, 2, dtype, 16)
    c = Cache(ops, [ctx], 1, seed=1)
    n = 300
    step = Step(c, [n], seed=2, spare=0)
    u = torch.sign(torch.randn(D, generator=torch.Generator().manual_seed(3))).cuda()
    ramp = torch.arange(n, device="cuda", dtype=torch.float32) * (8.0 / D)          # score / position: 8 D^-1/2, ~1 per token
    step.k[:, 0] = (u * ramp[:, None]).to(dtype)
    sign = {"rising": torch.ones(n), "falling": -torch.ones(n), "both": 1.0 - 2.0 * (torch.arange(n) % 2)}[order].cuda()
    step.q[:] = (u * sign[:, None, None]).to(dtype)
    want, bound = step.reference(None, 0)
    for n_splits in (1, 2):
        check(step.run(None, 0, n_splits), want, bound, dtype, f"{order} scores, ctx {ctx}, splits {n_splits}")


@pytest.mark.parametrize("D,bits,G,dtype,P,window,sinks", [(128, 8, 4, torch.float16, 16, 300, 16), (128, 4, 4, torch.bfloat16, 32, None, 0),
                                                            (64, 8, 1, torch.bfloat16, 16, 129, 5)])
def test_chunk_many_passes_agree(D, bits, G, dtype, P, window, sinks):
    """Passes in a row without a wait between them, on two steps in turn: the same bits every time, no wait given up."""
    from kushkash_b200 import _cuda
    ops = ops_of(D, bits, G, dtype, P)
    c = Cache(ops, [1300, 0, 517, 2000], 4, seed=bits)
    if window is not None:
        c.hide(c.lens, window, sinks)
    steps = [Step(c, [300, 130, 5, 77], seed=s, spare=0) for s in (1, 2)]
    want = [s.run(window, sinks) for s in steps]
    outs = []
    for i in range(200):
        s = steps[i % 2]
        outs.append(torch.empty_like(want[0]))
        ops.attend_chunk(s.q, s.k, s.v, outs[-1], s.qsl, s.seq_lens, c.tail_idx, c.pool, c.block_table, c.tail_k, D ** -0.5,
                         window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))
    assert _cuda.device_error() == 0


def test_chunk_in_place_and_negative_scale():
    """out may be q itself; a negative scale attends to the smallest products."""
    ops = ops_of(128, 4, 4, torch.bfloat16, 16)
    c = Cache(ops, [200], 2, seed=12)
    s = Step(c, [150], seed=3, spare=0)
    args = (s.qsl, s.seq_lens, c.tail_idx, c.pool, c.block_table, c.tail_k)
    q, want, neg = s.q.contiguous(), torch.empty(150, 8, 128, dtype=torch.bfloat16, device="cuda"), None
    ops.attend_chunk(q, s.k, s.v, want, *args, 0.07)
    neg = torch.empty_like(want)
    ops.attend_chunk(-q, s.k, s.v, neg, *args, -0.07)
    ops.attend_chunk(q, s.k, s.v, q, *args, 0.07)
    torch.cuda.synchronize()
    assert torch.equal(neg, want) and torch.equal(q, want)


def test_chunk_row_bounds_beyond_the_rows():
    """A query_start_loc that runs past the rows: only rows that are there are read and written."""
    ops = ops_of(128, 4, 4, torch.bfloat16, 16)
    c = Cache(ops, [64, 32], 1, seed=2)
    s = Step(c, [8, 12], seed=4, spare=0)
    want = s.run()
    out = torch.full((20, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.attend_chunk(s.q, s.k, s.v, out, torch.tensor([0, 8, 500], dtype=torch.int32, device="cuda"), s.seq_lens, c.tail_idx,
                     c.pool, c.block_table, c.tail_k, 128 ** -0.5)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_chunk_empty_step():
    ops = ops_of(128, 4, 4, torch.bfloat16, 16)
    c = Cache(ops, [20, 0], 1, seed=8)
    step = Step(c, [0, 0], seed=1)
    assert step.run().numel() == 0                                             # spare rows untouched (checked in run)
    assert step.run(n_splits=2).numel() == 0


def test_chunk_refusals():
    ops = ops_of(128, 4, 4, torch.bfloat16, 16)
    c = Cache(ops, [20], 1, seed=8)
    s = Step(c, [4], seed=1, spare=0)
    out = torch.empty(4, 4, 128, dtype=torch.bfloat16, device="cuda")
    good = dict(q=s.q, k=s.k, v=s.v, out=out, query_start_loc=s.qsl, seq_lens=s.seq_lens, tail_idx=c.tail_idx, cache=c.pool,
                block_table=c.block_table, tail_k=c.tail_k, scale=0.1)
    ops.attend_chunk(**good)
    odd = torch.empty(4 * 512 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 4, 128)
    for bad in (dict(q=s.q.float()), dict(k=s.k[:3]), dict(v=s.v[:, :, :64]), dict(out=out[:, :2]), dict(window=0), dict(sinks=1),
                dict(window=3, sinks=-1), dict(n_splits=2), dict(n_splits=2, work=torch.empty(10, device="cuda")),
                dict(query_start_loc=s.qsl.long()), dict(seq_lens=s.seq_lens.repeat(2)), dict(tail_k=c.tail_k[:, :, :8]),
                dict(q=odd), dict(n_splits=0), dict(q=s.q.cpu()), dict(block_table=c.block_table.cpu()),
                dict(n_splits=2, work=torch.empty(1 << 16))):
        with pytest.raises(ValueError):
            ops.attend_chunk(**{**good, **bad})

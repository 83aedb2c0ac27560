"""Chunk attention and the windowed decode at the edges of what their arguments allow."""
import pytest
import torch

from attend_ref import Cache, check, dequantize
from test_gpu_attend import Step, ops_of
from tolerance import half_ulp

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


def exact_rows(q, k, v, scale, seen, up):
    """softmax(q k) v of one head in 64 bits, and the bound of a kernel that takes these operands exactly (bf16 or fp16 values
    within fp16's normal range), adds scores in fp32 (D terms and the scale: D + 16 roundings) and rounds weights to fp16
    twice at most: 2^-11 relative each, or 2^-25 of a unit that is 2^up below the largest weight."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    s = (q @ k.T * scale).masked_fill(~seen, -torch.inf)
    ds = ((q.abs() @ k.abs().T) * abs(scale) * (q.shape[1] + 16) * 2.0 ** -24).masked_fill(~seen, 0).amax(-1)
    w = torch.softmax(s, dim=-1)
    small = (seen.double() @ v.abs()) * (2 * 2.0 ** -25 * 2.0 ** -up * w.amax(-1))[:, None]
    return w @ v, (w @ v.abs()) * (2 * 2.0 ** -11 + 2 * ds[:, None] + 2.0 ** -20) + small


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("n,at,window", [(100, 40, None), (100, 0, None), (300, 200, None), (3000, 0, None), (3000, 1, 2000), (1500, 1400, None)])
@pytest.mark.parametrize("gap", [8.0, 14.0, 17.3, 18.5])
def test_small_weights_beside_one_large_one(dtype, D, n, at, window, gap):
    """One token scores `gap` above all others and has the value zero (an attention sink): the output is made of the
    small weights, wherever in the tiles the large one stands."""
    ops = ops_of(D, 4, 1, dtype, 16)
    c = Cache(ops, [0], 1, seed=1)
    g = torch.Generator().manual_seed(n + at)
    side = torch.sign(torch.randn(D, generator=g))
    k = 0.05 * torch.randn(n, 1, D, generator=g)
    v = 0.5 + torch.rand(n, 1, D, generator=g)
    q = (1.0 + torch.rand(n, 1, D, generator=g)) * side
    scale = D ** -0.5
    k[at, 0] = side * gap / (1.5 * D * scale)
    v[at] = 0.0
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    qsl, lens = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, n], [n]))
    rows = torch.arange(max(at, n - 70), n)
    j = torch.arange(n)
    seen = j[None] <= rows[:, None]
    if window is not None:
        seen &= (j[None] > rows[:, None] - window) | (j[None] < at + 1)
    want, bound = exact_rows(q[rows, 0], k[:, 0], v[:, 0], scale, seen, 9)
    for n_splits in (1, 3):
        work = torch.full((ops.chunk_work_size(n, 1, n_splits),), float("nan"), device="cuda")
        out = torch.empty_like(q)
        ops.attend_chunk(q, k, v, out, qsl, lens, c.tail_idx, c.pool, c.block_table, c.tail_k, scale, n_splits, work, window=window,
                         sinks=at + 1 if window else 0)
        # (element by element, without check()'s relative norm: an fp16 output of 100 e^-18.5 = 9e-7 has a half step of 2^-25, 3%)
        got = out[rows, 0].double().cpu()
        worst = ((got - want).abs() / (bound + half_ulp(want.abs() + bound, dtype))).max().item()
        print(f"gap {gap} at {at} of {n} splits {n_splits}: {worst:.3f} of the bound")
        assert worst <= 1.0, f"{worst:.2f} times the bound"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,bits,P,ctx,new,window,sinks", [(128, 4, 16, 70, 12, None, 0), (128, 8, 32, 300, 200, None, 0),
                                                           (64, 4, 16, 128, 140, None, 0), (64, 8, 32, 261, 30, 100, 3),
                                                           (128, 8, 16, 5, 40, None, 0), (128, 4, 16, 20, 5, 4, 3), (64, 8, 16, 40, 9, 3, 20)])
def test_new_and_unfinished_keys_enter_as_they_are(dtype, D, bits, P, ctx, new, window, sinks):
    """Finished pages whose keys lie about 4000 in two channels, before new rows that do not: the new rows' keys must not lose
    what a shift by the pages' bias would round off.  q takes the two channels with opposite signs, so that the scores of the
    history stay small."""
    ops = ops_of(D, bits, 2, dtype, P)
    c = Cache(ops, [ctx], 1, seed=7, pad_blocks=8)
    g = torch.Generator().manual_seed(ctx + new)
    k = torch.randn(ctx, 1, D, generator=g)
    k[:, :, 4:6] += 4000
    k, v = k.to(dtype).cuda(), torch.randn(ctx, 1, D, generator=g).to(dtype).cuda()
    qsl = torch.tensor([0, ctx], dtype=torch.int32, device="cuda")
    js, jp, _ = ops.write_jobs(qsl, c.seq_lens, ctx // P + 2)
    ops.write(k, v, qsl, c.seq_lens, c.tail_idx, js, jp, c.pool, c.block_table, c.tail_k)
    torch.cuda.synchronize()
    c.k_all, c.v_all, c.kb_all = dequantize(c.pool, D, bits, P)
    c.tail_cpu = c.tail_k.cpu()
    step = Step(c, [new], seed=3, spare=0)
    step.q[:, :, 4], step.q[:, :, 5] = 8.0, -8.0
    kh, vh = c.tokens(0)
    full = ctx // P * P
    K, V = torch.cat([kh, step.k.cpu().double()])[:, 0], torch.cat([vh, step.v.cpu().double()])[:, 0]
    first = 0 if sinks or window is None else (ctx - window + 1) // P * P
    ref = c.kb_all[int(c.table_cpu[0, first // P]), 0] if full else torch.zeros(D, dtype=torch.float64)
    pos, j = ctx + torch.arange(new), torch.arange(ctx + new)
    seen = j[None] <= pos[:, None]
    if window is not None:
        seen &= (j[None] > pos[:, None] - window) | (j[None] < sinks)
    q = step.q.cpu().double().transpose(0, 1).reshape(-1, D)                   # [2 heads, rows]
    see = seen.repeat(2, 1)
    w = torch.softmax((q @ K.T * D ** -0.5).masked_fill(~see, -torch.inf), -1)
    # the records' keys are rounded to fp16 three times after the shift (bias - ref, c ks + that, and q is exact); every score
    # adds D terms of the unshifted size in fp32 (the shift among them), twice
    ds = (q.abs() @ (K - ref).abs().T * 3 * 2.0 ** -11 * (j < full) + 2 * (q.abs() @ K.abs().T) * (D + 16) * 2.0 ** -24) * D ** -0.5
    ds = ds.masked_fill(~see, 0)
    # w_j e^d_j / sum_i w_i e^d_i with |d| <= ds is off by a factor of at most e^ds_j sum_i w_i e^ds_i; weights and values are
    # rounded twice and once to fp16
    move = ds.exp() * (w * ds.exp()).sum(-1, keepdim=True) * (1 + 3 * 2.0 ** -11) - 1
    bound = (w * move) @ V.abs()
    want, bound = ((x.view(2, new, D).transpose(0, 1)) for x in (w @ V, bound))
    for n_splits in (1, 2):
        check(step.run(window, sinks, n_splits), want, bound, dtype, f"ctx {ctx} + {new} splits {n_splits}")


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16), (128, torch.float32), (256, torch.bfloat16)])
def test_a_row_of_nan_stays_its_own(D, dtype):
    """A query of NaN gives a row of NaN, split or not, and no other row changes."""
    ops = ops_of(D, 4, 2, dtype, 16)
    c = Cache(ops, [600], 2, seed=9)
    step = Step(c, [40], seed=1, spare=0)
    for n_splits in (1, 3):
        want = step.run(None, 0, n_splits)
        q = step.q.clone()
        step.q[7, 1] = float("nan")
        got = step.run(None, 0, n_splits)
        step.q.copy_(q)
        assert got[7, 1].isnan().all()
        got[7, 1] = want[7, 1]
        assert torch.equal(got, want)


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_two_streams_at_once(D, dtype):
    """Chunk attention on two streams and the windowed decode beside them, with work buffers of their own: the same bits as one
    after the other (blocks of two launches share an SM's tensor memory)."""
    from kushkash_b200 import _cuda
    ops = ops_of(D, 4, 4, dtype, 16)
    c = Cache(ops, [900, 300, 1500], 4, seed=6)
    steps = [Step(c, [200, 5, 60], seed=s, spare=0) for s in (1, 2)]
    rows, dec = steps[0].q.shape[0], torch.randn(3, 16, D, device="cuda").to(dtype)
    outs = [[torch.zeros(rows, 16, D, dtype=dtype, device="cuda") for _ in range(12)] for _ in steps]
    works = [torch.zeros(ops.chunk_work_size(rows, 4, 3), device="cuda") for _ in steps]
    outs.append([torch.zeros_like(dec) for _ in range(12)])

    def call(i, out):
        if i == 2:
            ops.decode(dec, out, c.pool, c.block_table, c.seq_lens, c.tail_idx, c.tail_k, D ** -0.5, window=700, sinks=4)
        else:
            s = steps[i]
            ops.attend_chunk(s.q, s.k, s.v, out, s.qsl, s.seq_lens, c.tail_idx, c.pool, c.block_table, c.tail_k, D ** -0.5, 3, works[i])

    want = [torch.zeros_like(o[0]) for o in outs]
    for i in range(3):
        call(i, want[i])
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for n in range(12):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                call(i, outs[i][n])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(3) for o in outs[i]) and _cuda.device_error() == 0

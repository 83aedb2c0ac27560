"""The windowed decode where a few tokens carry the weight and the others the output."""
import pytest
import torch

from attend_ref import Cache, dequantize
from test_gpu_window import ops_of, run
from tolerance import half_ulp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,bits,G,dtype,P", [(128, 8, 4, torch.float16, 16), (128, 8, 4, torch.bfloat16, 32), (128, 4, 7, torch.bfloat16, 16),
                                              (64, 8, 1, torch.float16, 32), (64, 4, 12, torch.bfloat16, 32), (256, 8, 2, torch.bfloat16, 16),
                                              (128, 8, 2, torch.float32, 16)])
@pytest.mark.parametrize("gap", [6.0, 10.0, 13.0, 17.0])
@pytest.mark.parametrize("spread", [1.0, 64.0])
def test_values_beside_a_sink(D, bits, G, dtype, P, gap, spread):
    """The first token scores `gap` above all others and has the value zero: the output is what the others' small weights make of
    their values (each channel of one sign, magnitudes of tokens up to `spread` apart in either direction)."""
    ops = ops_of(D, bits, G, dtype, P)
    n, window = 2000 + P // 2, 1000
    c = Cache(ops, [n], 1, seed=1)
    g = torch.Generator().manual_seed(D + bits)
    side = torch.sign(torch.randn(D, generator=g))
    scale = D ** -0.5
    k = 0.05 * torch.randn(n, 1, D, generator=g)
    k[0, 0] = side * gap / (1.5 * D * scale)
    size = spread ** (2 * torch.rand(n, 1, 1, generator=g) - 1)
    v = size * torch.where(torch.arange(D) % 3 == 0, 1.0, -1.0)
    v[0] = 0.0
    q = ((1.0 + torch.rand(1, G, D, generator=g)) * side).to(dtype).cuda()
    qsl = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    js, jp, _ = ops.write_jobs(qsl, c.seq_lens, n // P + 2)
    ops.write(k.to(dtype).cuda(), v.to(dtype).cuda(), qsl, c.seq_lens, c.tail_idx, js, jp, c.pool, c.block_table, c.tail_k)
    torch.cuda.synchronize()
    c.k_all, c.v_all, c.kb_all = dequantize(c.pool, D, bits, P)
    c.tail_cpu = c.tail_k.cpu()
    K, V = (t[:, 0] for t in c.tokens(0))
    j = torch.arange(n)
    seen = (j >= n - window) | (j < 1)
    K, V, j = K[seen], V[seen], j[seen]
    ref = c.kb_all[int(c.table_cpu[0, 0]), 0]
    x = q[0].cpu().double()
    s = x @ K.T * scale
    w = torch.softmax(s, -1)
    u = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -11
    # a record's key is rounded three times after the shift by ref (bias - ref, code times scale plus that) and q once; scores
    # add D terms in fp32 (the shift among them)
    ds = (x.abs() @ ((K - ref).abs() * (j < n // P * P)[:, None]).T * 4 * u + 2 * (x.abs() @ (K.abs() + ref.abs()).T) * (D + 16) * 2.0 ** -24) * scale
    # weights: the exponential, and p * vs rounded once; below fp16's normal range in steps of 2^-25 of a unit that is at most
    # vs / 2^9 for the largest vs seen, times a code of at most 2^(bits - 1)
    move = ds.exp() * (w * ds.exp()).sum(-1, keepdim=True) * (1 + 2 * u + 2.0 ** -20) - 1
    vs = 2 * spread / (2 ** bits - 1) * 1.01
    small = 0.0 if dtype == torch.float32 else (w.amax(-1, keepdim=True) * len(j) * 2.0 ** -25 * 2.0 ** -9 * vs * 2 ** (bits - 1))
    want, bound = w @ V, (w * move) @ V.abs() + small
    for n_splits, fused in ((1, False), (3, False), (3, True)):
        got = run(c, q, window, 1, n_splits, fused)[0].double().cpu()
        worst = ((got - want).abs() / (bound + half_ulp(want.abs() + bound, dtype))).max().item()
        print(f"gap {gap} spread {spread} splits {n_splits}: {worst:.3f} of the bound, rel {((got - want).norm() / want.norm()).item():.2e}, "
              f"bound {(bound.norm() / want.norm()).item():.2e}")
        assert worst <= 1.0, f"splits {n_splits}: {worst:.2f} times the bound"


@pytest.mark.parametrize("D,bits,G,dtype,P,H,S", [(128, 4, 4, torch.bfloat16, 16, 2, 5), (128, 8, 7, torch.float16, 32, 1, 3),
                                                  (64, 8, 1, torch.bfloat16, 16, 1, 1), (256, 4, 3, torch.float16, 32, 1, 1),
                                                  (64, 4, 3, torch.float32, 16, 1, 3), (128, 4, 20, torch.bfloat16, 16, 1, 2)])
@pytest.mark.parametrize("n_splits", [2, 3, 7, 33])
@pytest.mark.parametrize("rotate", [False, True])
def test_merges_agree(D, bits, G, dtype, P, H, S, n_splits, rotate):
    """The merge in the decode launch and the one behind it give the same bits, wherever the partials lie in the work buffer."""
    ops = ops_of(D, bits, G, dtype, P)
    c = Cache(ops, [900, 33, 0, 411, 1200][:S], H, seed=3)
    q = torch.randn(S, H * G, D, generator=torch.Generator().manual_seed(n_splits)).to(dtype).cuda()
    got = [run(c, q, 700, 20, n_splits, fused, rotate=rotate) for fused in (False, True)]
    assert not got[0].isnan().any() and torch.equal(*got)

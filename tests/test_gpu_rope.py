"""Rotary positions against the definition in 64 bits: layouts, parts of the head, scalings, strides, far positions."""
import math

import pytest
import torch

from tolerance import half_ulp

pytestmark = pytest.mark.gpu
SCALINGS = [None, {"rope_type": "linear", "factor": 4.0}, {"rope_type": "ntk", "factor": 4.0},
            {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 8192},
            {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_max_position_embeddings": 8192}]


def ops_of(D, dtype):
    from kushkash_b200 import Ops
    return Ops(torch.device("cuda:0"), D, 4, 4, dtype, 32)


def rotate(x, pos, r, theta, inter, scaling):
    """(rotated rows in 64 bits, sum of the magnitudes that meet in each output)"""
    from kushkash_b200 import rotary_frequencies
    freq, factor = rotary_frequencies(r, theta, scaling)
    a = torch.tensor([[math.remainder(float(p) * f, 2 * math.pi) for f in freq] for p in pos.tolist()], dtype=torch.float64)
    c, s = (factor * a.cos())[:, None], (factor * a.sin())[:, None]
    x = x.double().cpu()
    y, mass = x.clone(), x.abs()
    i, j = (slice(0, r, 2), slice(1, r, 2)) if inter else (slice(0, r // 2), slice(r // 2, r))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    mass[..., i] = mass[..., j] = factor * (x[..., i].abs() + x[..., j].abs())
    return y, mass


def check(got, x, pos, r, theta, inter, scaling, dtype):
    want, mass = rotate(x, pos, r, theta, inter, scaling)
    # the reference's own angle: |pos| f in 64 bits, off by up to half an ulp of a double; the kernel's: a rounding of the
    # half-turn fraction to fp32 (2^-25 pi), sincospif (2 ulp), the factor, two products and their sum: 8 u in all
    angle = 2.0 ** -53 * (pos.abs().max().item() + 1)
    bound = mass * (8 * 2.0 ** -24 + 2 * angle)
    err = (got.double().cpu() - want).abs()
    assert (err <= bound + half_ulp(want.abs() + bound, dtype)).all(), float((err - bound).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,r,inter", [(64, 64, False), (64, 64, True), (128, 128, False), (128, 64, True), (128, 20, False),
                                       (128, 2, True), (256, 256, False), (256, 128, True), (64, 6, True)])
def test_rope(dtype, D, r, inter):
    ops = ops_of(D, dtype)
    g = torch.Generator().manual_seed(D + r)
    for n, scaling, high in zip((1, 3, 50, 1300, 77), SCALINGS, (10, 5000, 1 << 20, 40000, 1 << 31)):
        if scaling and scaling["rope_type"] == "ntk" and r == 2:
            continue
        H, Hq = 2, 5
        qkv = torch.randn(n, (Hq + 2 * H) * D, generator=g).to(dtype).cuda()
        q, k = qkv[:, :Hq * D].view(n, Hq, D), qkv[:, Hq * D:(Hq + H) * D].view(n, H, D)
        pos = torch.randint(0, high, (n,), generator=g, dtype=torch.int64)
        pos[-1] = high - 1
        plan = ops.rotary(r, 500000.0, interleaved=inter, scaling=scaling)
        q2, k2 = ops.rope(q, k, pos.cuda() if high > 5000 else pos.to(torch.int32).cuda(), plan)
        for got, x in ((q2, q), (k2, k)):
            check(got, x, pos, r, 500000.0, inter, scaling, dtype)
            assert torch.equal(got[..., r:], x[..., r:])
        copy = qkv.clone()                                                     # in place, inside packed rows
        qc, kc = copy[:, :Hq * D].view(n, Hq, D), copy[:, Hq * D:(Hq + H) * D].view(n, H, D)
        ops.rope(qc, kc, pos.cuda(), plan, qc, kc)
        assert torch.equal(qc, q2) and torch.equal(kc, k2)
        assert torch.equal(copy[:, (Hq + H) * D:], qkv[:, (Hq + H) * D:])      # v untouched


def test_rope_odd_alignment_and_strides():
    """Rows that 16-byte vectors do not divide, heads apart, one of q and k alone, negative and 64-bit positions."""
    ops = ops_of(128, torch.bfloat16)
    plan = ops.rotary(64)
    base = torch.randn(9, 3, 131).to(torch.bfloat16).cuda()
    pos = torch.tensor([0, -1, 7, 1 << 40, -(1 << 33), 3, 2, 1, 12345])
    x = base[:, :, 3:]
    y = torch.zeros(9, 3, 133, dtype=torch.bfloat16, device="cuda")
    got, none = ops.rope(x, None, pos.cuda(), plan, y[:, :, 5:])
    assert none is None and (y[:, :, :5] == 0).all()
    near = pos.abs() < (1 << 20)
    check(got[near], x[near], pos[near], 64, 10000.0, False, None, torch.bfloat16)
    # the reference's frequency in 64 bits is off by 2^-53 relative: 2^-13 of a radian at 2^40
    want, mass = rotate(x[~near], pos[~near], 64, 10000.0, False, None)
    err = (got[~near].double().cpu() - want).abs()
    assert (err <= mass * 2 * 2.0 ** -12 + half_ulp(want.abs(), torch.bfloat16) * 1.01).all()
    only_k = ops.rope(None, x, pos.cuda(), plan)[1]
    assert torch.equal(only_k, got)


def test_rope_empty_and_large():
    ops = ops_of(128, torch.float16)
    plan = ops.rotary()
    e = torch.empty(0, 4, 128, dtype=torch.float16, device="cuda")
    assert ops.rope(e, e, torch.empty(0, dtype=torch.int64, device="cuda"), plan)[0].shape == e.shape
    n = 420001                                                                 # more than 2^31 channels
    q = torch.randn(n, 40, 128, device="cuda", dtype=torch.float16)
    pos = torch.arange(n, device="cuda")
    got = ops.rope(q, None, pos, plan)[0]
    at = [0, 1, n // 2, n - 1]
    check(got[at], q[at], pos[at].cpu(), 128, 10000.0, False, None, torch.float16)


def test_rope_graph_and_stream():
    ops = ops_of(128, torch.bfloat16)
    plan = ops.rotary(interleaved=True)
    q, k = (torch.randn(5, h, 128, device="cuda").to(torch.bfloat16) for h in (8, 2))
    pos, qo, ko = torch.arange(5, device="cuda"), torch.empty_like(q), torch.empty_like(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rope(q, k, pos, plan, qo, ko)
    pos += 100
    graph.replay()
    torch.cuda.synchronize()
    want = ops.rope(q, k, pos, plan)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


def test_rope_refusals():
    ops = ops_of(128, torch.bfloat16)
    plan = ops.rotary()
    q = torch.randn(4, 2, 128, device="cuda").to(torch.bfloat16)
    pos = torch.arange(4, device="cuda")
    other = ops_of(64, torch.bfloat16).rotary()
    for args in ((q.float(), None, pos, plan), (q, None, pos[:3], plan), (q, None, pos.float(), plan), (q[..., :64], None, pos, plan),
                 (q, None, pos, other), (None, None, pos, plan, q), (q, None, pos, plan, q[:, :1]),
                 (q.cpu(), None, pos, plan), (q, None, pos.cpu(), plan), (q, q.cpu(), pos, plan), (q.transpose(1, 2), None, pos, plan), (q, None, pos.repeat(2)[::2], plan)):
        with pytest.raises(ValueError):
            ops.rope(*args)
    for bad in (3, 0, 130):
        with pytest.raises(ValueError):
            ops.rotary(bad)

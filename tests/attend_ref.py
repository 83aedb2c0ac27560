"""Attention over a paged cache from its definition, in 64 bits on the CPU, and the error that a kernel's own roundings
allow: what the tests of the windowed decode and of chunk attention compare with.

The bound of an output element follows the roundings one by one.  With u the unit roundoff of the type a kernel feeds
its products (fp16 2^-11, fp32 2^-24 times the terms a dot product adds), w_j the exact softmax weights:
  score   |d s_j| <= scale * sum_d |q_d| (|k_jd| + 2 |ref_d|) * c_s u   (operands rounded to the type; ref = the key
          bias that a kernel subtracts from every key before it rounds, 0 if it subtracts none), so a weight moves by at
          most 2 max|d s| relative (its own and the sum's)
  weight  one rounding, value: one rounding of c * vs + v_b                                  -> 2 u
so |d o| <= sum_j w_j |v_j| (2 u + 2 max_j |d s_j|), and the output's own rounding: half an ulp.
"""
import torch

from tolerance import BOUNDS, half_ulp


def dequantize(pool: torch.Tensor, D: int, bits: int, P: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Records [blocks, H, RB] -> K, V [blocks, H, P, D] and the key biases [blocks, H, D], fp64."""
    raw = pool.cpu()
    dc = D if bits == 8 else D // 2
    codes = raw[..., :2 * P * dc].reshape(*raw.shape[:2], 2, P, dc)
    if bits == 8:
        c = codes.contiguous().view(torch.int8).double()
    else:
        c = torch.cat([codes & 15, codes >> 4], dim=-1).double()
        c = c - 16 * (c > 7)
    s = raw[..., 2 * P * dc:].contiguous().view(torch.float16).double()
    ks, kb, vs, vb = s.split([D, D, P, P], dim=-1)
    return c[:, :, 0] * ks[:, :, None] + kb[:, :, None], c[:, :, 1] * vs[..., None] + vb[..., None], kb


def attend(q, k, v, pos_q, pos_k, scale, window=None, sinks=0, ref=None, u=2.0 ** -11, c_s=1.0):
    """q [T, H, G, D], k, v [N, H, D], positions [T], [N] -> (out [T, H, G, D], bound of its error before rounding)."""
    q, k, v = q.double(), k.double(), v.double()
    see = pos_k[None] <= pos_q[:, None]
    if window is not None:
        see &= (pos_k[None] > pos_q[:, None] - window) | (pos_k[None] < sinks)
    see = see[:, None, None]
    s = torch.einsum("thgd,nhd->thgn", q, k) * scale
    mass = k.abs() if ref is None else k.abs() + 2 * ref.double().abs()
    ds = (torch.einsum("thgd,nhd->thgn", q.abs(), mass) * abs(scale) * c_s * u).masked_fill(~see, 0).amax(-1)
    w = torch.softmax(s.masked_fill(~see, -torch.inf), dim=-1)
    out = torch.einsum("thgn,nhd->thgd", w, v)
    bound = torch.einsum("thgn,nhd->thgd", w, v.abs()) * (2 * u + 2 * ds[..., None])
    return out, bound


def check(got, want, bound, dtype, what):
    got = got.detach().double().cpu()
    assert not torch.isnan(got).any(), f"{what}: NaN"
    err = (got - want).abs()
    allow = bound + half_ulp(want.abs() + bound, dtype)
    worst = float((err / allow.clamp(min=1e-30)).max()) if err.numel() else 0.0
    rel = float((got - want).norm() / want.norm().clamp(min=1e-30)) if err.numel() else 0.0
    print(f"[attend] {what}: {worst:.3f} of the bound, rel-norm {rel:.2e}")
    assert worst <= 1.0, f"{what}: error {worst:.2f} times the bound, rel-norm {rel:.2e}"
    assert rel <= BOUNDS[dtype][1], f"{what}: rel-norm {rel:.2e} above the decode's bound"


class Cache:
    """A cache of ragged sequences written through ops.write, and its 64-bit content.  Every byte that no token wrote is
    poison (NaN scales, NaN tail rows), and `hide` points the table entries of unseen pages at a poisoned block."""

    def __init__(self, ops, lens, H, seed, pad_blocks=3, strided=False):
        dev, D, P, bits, dt = ops.device, ops.D, ops.P, ops.bits, ops.dtype
        self.ops, self.lens, self.H, S = ops, list(lens), H, len(lens)
        g = torch.Generator().manual_seed(seed)
        from kushkash_b200 import record_bytes
        rb = record_bytes(D, bits, P)
        pages = [-(-n // P) for n in lens]
        blocks = sum(pages) + pad_blocks
        raw = torch.full((blocks, H * rb + (48 if strided else 0)), 0xFF, dtype=torch.uint8, device=dev)
        self.pool = raw[:, :H * rb].view(blocks, H, rb)
        perm = torch.randperm(blocks - 1, generator=g) + 1                     # block 0 stays poison
        table = torch.zeros(S, max(pages + [1]) + 2, dtype=torch.int32)
        at = 0
        for s, n in enumerate(pages):
            table[s, :n] = perm[at:at + n]
            at += n
        self.block_table = table.to(dev)
        self.tail_k = torch.full((S + 1, H, P, D), float("nan"), dtype=dt, device=dev)
        self.tail_idx = (torch.randperm(S + 1, generator=g)[:S]).to(torch.int32).to(dev)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        off = 2 * torch.randn(H, D, generator=g)
        off[:, 1] += 15
        rows = sum(lens)
        K = (torch.randn(rows, H, D, generator=g) + off).to(dt)
        V = torch.randn(rows, H, D, generator=g).to(dt)
        if rows:
            qsl = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(dev)
            js, jp, _ = ops.write_jobs(qsl, self.seq_lens, rows // P + 2 * S)
            ops.write(K.to(dev), V.to(dev), qsl, self.seq_lens, self.tail_idx, js, jp, self.pool, self.block_table, self.tail_k)
            torch.cuda.synchronize()
        self.k_all, self.v_all, self.kb_all = dequantize(self.pool, D, bits, P)
        self.table_cpu, self.tail_cpu, self.tidx_cpu = table, self.tail_k.cpu(), self.tail_idx.cpu()

    def tokens(self, s):
        """K, V [n, H, D] of sequence s and its first key bias."""
        P, n = self.ops.P, self.lens[s]
        t = torch.arange(n)
        blk = self.table_cpu[s].long()[t // P]
        k, v = self.k_all[blk, :, t % P], self.v_all[blk, :, t % P]
        full = n // P * P
        if n > full:
            k[full:] = self.tail_cpu[int(self.tidx_cpu[s])].double().transpose(0, 1)[:n - full]
        return k, v

    def hide(self, first_pos, window, sinks):
        """Point the table entries of pages that queries from first_pos[s] on do not see at the poisoned block."""
        P, t = self.ops.P, self.table_cpu.clone()
        for s, n in enumerate(self.lens):
            lo = max(0, first_pos[s] - window + 1)
            for p in range(-(-n // P)):
                if p * P >= min(sinks, lo) and (p + 1) * P <= lo:
                    t[s, p] = 0
        self.block_table.copy_(t)

    def ref(self, s, page=0):
        n = self.lens[s]
        return self.kb_all[int(self.table_cpu[s, page])].abs() if n >= self.ops.P else None

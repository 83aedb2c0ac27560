"""kushkash_b200.Ops: the library's own PyTorch-facing operator object, one per (device, head_dim, bits, group,
dtype, page), calling the C ABI of libkush_sm100.so (include/kushkash_b200.h) directly.

Two ways reach the same kernels:
  * the reference's own operator layer (kushkash/_ops.py Ops, cache.py KushCache, the HF / vLLM / SGLang
    integrations), unchanged, through the drop-in loader kushkash_b200._cuda (kushkash_b200.dropin.install());
  * this class, which the benchmarks, the sharding layer and the parity tests use.  Its calls take the same
    tensors with the same meaning as kushkash.Ops (kushkash/_ops.py:42-213) -- so code written against one reads
    the same against the other -- plus what the reference cannot express: the page size (16 or 32 tokens), the
    rotation fused into the kernels, a decode launch order and the split-KV partials without their combine.

Tensor conventions (the record layout of kushkash/kush/quant.mojo:53-87):
  cache        [blocks, H, ...] uint8 (any view whose (block, head) records are contiguous; byte strides are passed)
  tail_k       [slots, H, P, D] in the kernel dtype: exact K of each sequence's unfinished page (slot tail_idx[s])
  k, v rows    [rows, H, D], row strides free, head stride D
  q, out       [S, H * G, D] contiguous, q head = kv_head * G + g
  index tensors int32 on the device

Every call is asynchronous on torch's current stream of the device; nothing allocates except the optional outputs
of fwht() and longest_first().  There is no CPU path and no PyTorch fallback: a non-CUDA device, a missing library
or an unsupported configuration raises.
"""
from __future__ import annotations

import functools
import os

import torch

from . import _cuda
from ._build import PAGE, GpuConfig
from ._rotary import Rotary, make_rotary

_DTYPE_NAMES = {torch.float16: "float16", torch.bfloat16: "bfloat16", torch.float32: "float32"}
MAX_SPLITS = 256
MIN_SPLIT_PAGES = 16
LONG_SPLIT_PAGES = 100
CHUNK_TILE = 256
MIN_CHUNK_SPLIT = 256
MIN_SIMT_SPLIT = 160
MIN_SIMT_CHUNK_SPLIT = 48
_I32_MAX = 2 ** 31 - 1


def record_bytes(head_dim: int, bits: int, page: int = PAGE) -> int:
    """Bytes of one (page, kv head) record: P code rows each for K and V (D bytes at 8 bits, D/2 at 4) and fp16
    K scale / bias per channel and V scale / bias per token (the format of kushkash/kush/quant.mojo:53-87)."""
    dc = head_dim if bits == 8 else head_dim // 2
    return 2 * page * dc + 4 * head_dim + 4 * page


def split_factor(num_seqs: int, num_kv_heads: int, max_full_pages: int, sms: int, ctas_per_sm: int = 4) -> int:
    """Split-KV factor: enough splits that the decode grid fills the ~ctas_per_sm resident CTAs of every SM once (any
    integer, not only powers of two), at most MAX_SPLITS and at least MIN_SPLIT_PAGES pages per split; 1 when the
    (sequence, kv head) units alone fill half the GPU.  (The reference grows powers of two up to 32 while the grid
    has fewer than 6 blocks per SM, kushkash/_ops.py:182-189; on B200 fewer, fuller splits measured faster: per-split
    setup, merge and the combine grow with the split count -- 8 sequences x 4 kv heads x 64 pages decode fastest at 4
    splits, not 16.)"""
    units, cap = num_seqs * num_kv_heads, ctas_per_sm * sms
    if units == 0 or units * 2 >= cap or max_full_pages < 8:
        return 1
    ns = max(1, min(MAX_SPLITS, cap // units, max_full_pages // MIN_SPLIT_PAGES))
    # Past two CTAs per SM, splits of fewer than LONG_SPLIT_PAGES pages lose more to per-split setup and merge than
    # the extra CTAs give back (config 4 geometry with 2 kv heads: 74 splits of 55 pages 65.7 us, 37 of 111 56.1 us;
    # with 4 kv heads 37 splits of 111 pages stay the fastest): keep two CTAs per SM and splits of ~LONG_SPLIT_PAGES.
    if units * ns > 2 * sms and max_full_pages // ns < LONG_SPLIT_PAGES:
        ns = max(-(-2 * sms // units), min(ns, -(-max_full_pages // LONG_SPLIT_PAGES)))
    return ns


def chunk_split_factor(num_rows: int, num_seqs: int, num_kv_heads: int, group: int, max_len: int, sms: int) -> int:
    """Split factor of attend_chunk(): its blocks are one per (tile of CHUNK_TILE query rows, kv head); when they fill less
    than half the SMs the keys of each are divided so that the SMs are filled once, with at least MIN_CHUNK_SPLIT tokens
    a split and at most MAX_SPLITS of them."""
    units = max(1, max(num_seqs, -(-num_rows * group // CHUNK_TILE)) * num_kv_heads)
    return max(1, min(MAX_SPLITS, sms // units, max_len // MIN_CHUNK_SPLIT))


def _pool(cache: torch.Tensor) -> tuple[int, int, int]:
    """(address, block stride, head stride) of a record pool, strides in bytes."""
    e = cache.element_size()
    return cache.data_ptr(), cache.stride(0) * e, cache.stride(1) * e


def _table(block_table: torch.Tensor) -> tuple[int, int]:
    """(address, row stride in entries) of a block table."""
    return block_table.data_ptr(), block_table.stride(0)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class Ops:
    """The kernels of one (device, head_dim, bits, group, dtype, page) configuration."""

    def __init__(self, device: torch.device, head_dim: int, bits: int, group: int, dtype: torch.dtype,
                 page: int = PAGE):
        device = torch.device(device)
        _need(device.type == "cuda", "kushkash_b200 runs on CUDA (B200, sm_100a) devices only; it has no CPU path")
        _need(head_dim in (64, 128, 256), "GPU head_dim must be 64, 128 or 256")
        _need(dtype in _DTYPE_NAMES, f"dtype must be one of {tuple(_DTYPE_NAMES)}")
        self.dev = device.index if device.index is not None else torch.cuda.current_device()
        self.device = torch.device("cuda", self.dev)
        self.D, self.bits, self.G, self.dtype, self.P = head_dim, bits, group, dtype, page
        self.cfg = GpuConfig(head_dim, bits, group, _DTYPE_NAMES[dtype], _cuda.arch(self.dev), page)
        self.sms = _cuda.sm_count(self.dev)
        self.lib = _cuda.lib()
        self._fmt = (head_dim, bits, page, self.cfg.dtype_code)        # leading arguments of most entry points
        self.fused_write = os.environ.get("KUSHKASH_FUSED_WRITE", "1") != "0"

    def _run(self, entry: str, *args) -> None:
        """Call one C entry point with torch's current stream of this device appended; raise on a failed status."""
        fn = getattr(self.lib, entry)
        if torch._C._cuda_getDevice() == self.dev:           # (CUDA is up since __init__)
            rc = fn(*args, _cuda.raw_stream(self.dev))
        else:
            with torch.cuda.device(self.dev):
                rc = fn(*args, _cuda.raw_stream(self.dev))
        _cuda.check(rc, entry)

    def _here(self, what: str, *tensors: torch.Tensor) -> None:
        """Refuse tensors of another device: their addresses would fault in a kernel."""
        for t in tensors:
            if t.get_device() != self.dev:
                raise ValueError(f"{what}: every tensor must be on {self.device}, got one on {t.device}")

    # ---------------------------------------------------------------- quantize-on-write
    def append(self, k: torch.Tensor, v: torch.Tensor, seq_lens: torch.Tensor, tail_idx: torch.Tensor,
               cache: torch.Tensor, block_table: torch.Tensor, tail_k: torch.Tensor, pos_offset: int, advance: bool,
               *, rotate: bool = False) -> None:
        """One new token per sequence: row s of k / v lands at position seq_lens[s] + pos_offset (negative positions
        are skipped); advance stores pos + 1 into seq_lens.  rotate: rotate the rows first (canonical Walsh-Hadamard,
        bit for bit what fwht() then append() store)."""
        entry = "kush_sm100_append_rotated" if rotate else "kush_sm100_append"
        self._run(entry, *self._fmt, k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), seq_lens.data_ptr(),
                  int(pos_offset), int(bool(advance)), tail_idx.data_ptr(), *_pool(cache), tail_k.data_ptr(),
                  *_table(block_table), k.shape[1], k.shape[0])

    def write(self, k: torch.Tensor, v: torch.Tensor, query_start_loc: torch.Tensor, seq_lens: torch.Tensor,
              tail_idx: torch.Tensor, job_seq: torch.Tensor, job_page: torch.Tensor, cache: torch.Tensor,
              block_table: torch.Tensor, tail_k: torch.Tensor) -> None:
        """Ragged multi-token write: sequence s owns rows [qsl[s], qsl[s+1]) at the positions that end at
        seq_lens[s] (which already counts them); job j is logical page job_page[j] of sequence job_seq[j].  One
        launch (mode 2); KUSHKASH_FUSED_WRITE=0 (or fused_write = False) runs the two-launch form (modes 0, 1)."""
        n_jobs = job_seq.numel()
        if n_jobs == 0:
            return
        for mode in ((2,) if self.fused_write else (0, 1)):
            self._run("kush_sm100_write", *self._fmt, k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0),
                      query_start_loc.data_ptr(), seq_lens.data_ptr(), tail_idx.data_ptr(), job_seq.data_ptr(),
                      job_page.data_ptr(), mode, *_pool(cache), tail_k.data_ptr(), *_table(block_table), k.shape[1],
                      n_jobs)

    def write_jobs(self, query_start_loc: torch.Tensor, seq_lens: torch.Tensor, max_jobs: int,
                   job_seq: torch.Tensor | None = None, job_page: torch.Tensor | None = None,
                   n_jobs: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The jobs of write() for a step, built on the device (kush_sm100_write_jobs): one per (sequence, logical
        page its rows touch), in sequence then page order, then padding to max_jobs that write() skips.  Returns
        (job_seq, job_page, n_jobs) -- n_jobs a one-element device tensor.  max_jobs >= rows // P + 2 * S always
        suffices; nothing is read back to the host, so the call can be captured in a CUDA graph."""
        S = seq_lens.numel()
        _need(all(t.dtype == torch.int32 and t.is_contiguous() for t in (query_start_loc, seq_lens))
              and query_start_loc.numel() >= S + 1, "write_jobs: query_start_loc [S + 1] and seq_lens [S] must be "
              "contiguous int32")
        dev = seq_lens.device
        job_seq = torch.empty(max_jobs, dtype=torch.int32, device=dev) if job_seq is None else job_seq
        job_page = torch.empty(max_jobs, dtype=torch.int32, device=dev) if job_page is None else job_page
        n_jobs = torch.empty(1, dtype=torch.int32, device=dev) if n_jobs is None else n_jobs
        _need(job_seq.numel() >= max_jobs and job_page.numel() >= max_jobs and n_jobs.numel() >= 1,
              "write_jobs: output tensors smaller than max_jobs")
        self._run("kush_sm100_write_jobs", query_start_loc.data_ptr(), seq_lens.data_ptr(), S, self.P,
                  job_seq.data_ptr(), job_page.data_ptr(), max_jobs, n_jobs.data_ptr())
        return job_seq[:max_jobs], job_page[:max_jobs], n_jobs

    def unpack_plan(self, query_start_loc: torch.Tensor, seq_lens: torch.Tensor, tail_idx: torch.Tensor,
                    block_table: torch.Tensor, max_pages: int, max_tails: int, max_new: int) -> dict:
        """The plan of unpack() for a step that packs every sequence's history and new rows together (sequence s
        at rows kv_start[s] .. kv_start[s + 1]), built on the device (kush_sm100_unpack_plan); each list padded to
        its capacity with entries unpack() skips.  Returns kv_start [S + 1] (the varlen attention's cu_seqlens_k),
        page_blk, page_dst, tail_blk, tail_info, new_dst and counts [4] (full pages, partial pages, new rows, packed
        rows), all on the device."""
        S, dev = seq_lens.numel(), seq_lens.device
        _need(all(t.dtype == torch.int32 and t.is_contiguous() for t in (query_start_loc, seq_lens, tail_idx))
              and block_table.dtype == torch.int32 and block_table.stride(1) == 1,
              "unpack_plan: index tensors must be int32 (query_start_loc, seq_lens, tail_idx contiguous)")
        i32 = dict(dtype=torch.int32, device=dev)
        plan = dict(kv_start=torch.empty(S + 1, **i32), page_blk=torch.empty(max_pages, **i32),
                    page_dst=torch.empty(max_pages, **i32), tail_blk=torch.empty(max_tails, **i32),
                    tail_info=torch.empty(3 * max_tails, **i32), new_dst=torch.empty(max_new, **i32),
                    counts=torch.empty(4, **i32))
        self._run("kush_sm100_unpack_plan", query_start_loc.data_ptr(), seq_lens.data_ptr(), tail_idx.data_ptr(),
                  *_table(block_table), S, self.P, plan["kv_start"].data_ptr(), plan["page_blk"].data_ptr(),
                  plan["page_dst"].data_ptr(), max_pages, plan["tail_blk"].data_ptr(), plan["tail_info"].data_ptr(),
                  max_tails, plan["new_dst"].data_ptr(), max_new, plan["counts"].data_ptr())
        return plan

    # ---------------------------------------------------------------- rotation and unpack
    def fwht(self, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """The canonical Walsh-Hadamard rotation of every D-row of x (contiguous, this dtype) into out (a new
        tensor, or x itself, or any contiguous tensor of x's shape and dtype); returns out."""
        y = torch.empty_like(x) if out is None else out
        _need(x.dtype == self.dtype and y.dtype == self.dtype, f"fwht: tensors must be {self.dtype}")
        _need(x.is_contiguous() and y.is_contiguous() and x.shape == y.shape and x.shape[-1] == self.D,
              f"fwht: x and out must be contiguous, of one shape, with last dim {self.D}")
        rows = x.numel() // self.D
        if rows:
            self._run("kush_sm100_fwht", self.D, self.cfg.dtype_code, x.data_ptr(), y.data_ptr(), self.D, self.D,
                      rows)
        return y

    def unpack(self, cache: torch.Tensor, page_blk: torch.Tensor, page_dst: torch.Tensor, tail_blk: torch.Tensor,
               tail_info: torch.Tensor, tail_k: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
               new_dst: torch.Tensor, kp: torch.Tensor, vp: torch.Tensor, rot: bool) -> None:
        """Keys and values of a prefill with history into kp / vp ([rows, H, D], contiguous, this dtype): full pages
        (block page_blk[i] -> rows page_dst[i] + t), partial pages (block tail_blk[i], tail_info[i] = first row,
        tokens, tail slot; K from tail_k), new rows (row j of k_new / v_new -> row new_dst[j]); rot rotates history
        back.  Index values are not checked on the host (that would synchronise); the tensors' kinds are."""
        H = kp.shape[1]
        idx = (page_blk, page_dst, tail_blk, tail_info, new_dst)
        _need(all(t.dtype == torch.int32 and t.is_contiguous() for t in idx), "unpack: index tensors must be "
              "contiguous int32")
        _need(all(t.dtype == self.dtype for t in (tail_k, k_new, v_new, kp, vp)),
              f"unpack: tail_k, k_new, v_new, kp and vp must be {self.dtype}")
        _need(kp.shape == vp.shape and kp.dim() == 3 and kp.shape[2] == self.D and kp.is_contiguous()
              and vp.is_contiguous(), f"unpack: kp and vp must be contiguous [rows, H, {self.D}]")
        _need(all(t.dim() == 3 and tuple(t.shape[1:]) == (H, self.D) and t.stride(1) == self.D and t.stride(2) == 1
                  for t in (k_new, v_new)), "unpack: k_new / v_new rows must be [n, H, D] with head stride D")
        n_pages, n_tail, n_new = page_blk.numel(), tail_blk.numel(), new_dst.numel()
        _need(page_dst.numel() == n_pages and tail_info.numel() == 3 * n_tail
              and min(k_new.shape[0], v_new.shape[0]) >= n_new,
              "unpack: one page_dst per page, three tail_info ints per partial page, one k_new / v_new row per new_dst")
        if n_pages + n_tail + n_new == 0:
            return
        self._run("kush_sm100_unpack", *self._fmt, *_pool(cache), H, page_blk.data_ptr(), page_dst.data_ptr(),
                  n_pages, tail_blk.data_ptr(), tail_info.data_ptr(), n_tail, tail_k.data_ptr(), k_new.data_ptr(),
                  v_new.data_ptr(), k_new.stride(0), v_new.stride(0), new_dst.data_ptr(), n_new, kp.data_ptr(),
                  vp.data_ptr(), int(bool(rot)))

    # ---------------------------------------------------------------- rotary positions
    def rotary(self, rotary_dim: int | None = None, theta: float = 10000.0, *, interleaved: bool = False,
               scaling: dict | None = None) -> Rotary:
        """A plan for rope(): the first rotary_dim channels (default all) of a head turn, in pairs (i, i + r/2) or,
        interleaved, (2i, 2i + 1), with base frequencies theta^(-2i/r) and the long-context scaling of
        rotary_frequencies().  Made once (a small device tensor); good for every position."""
        return make_rotary(self.device, self.D, rotary_dim, theta, interleaved, scaling)

    def rope(self, q: torch.Tensor | None, k: torch.Tensor | None, positions: torch.Tensor, rotary: Rotary,
             q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None
             ) -> tuple[torch.Tensor | None, torch.Tensor | None]:
        """Rotary positions of the rows of a step, before append() / write() / attend_chunk(): q [rows, Hq, D] and k
        [rows, H, D] (either may be None; row and head strides free, e.g. parts of q|k|v rows), row i at positions[i]
        (int32 or int64, contiguous), into q_out and k_out (new tensors, or q and k themselves, or others of their
        shapes that overlap neither).  Returns (q_out, k_out).  Angles are exact to fp32 for every position; one rounding to the dtype."""
        D, rows, dt = self.D, positions.shape[0] if positions.dim() == 1 else -1, self.dtype
        wide = positions.dtype == torch.int64
        if rows < 0 or not (wide or positions.dtype == torch.int32) or not positions.is_contiguous():
            raise ValueError("rope: positions must be a contiguous row of int32 or int64")
        self._here("rope", positions, *(t for t in (q, k, q_out, k_out) if t is not None))
        if rotary.head_dim != D or rotary.turns.device != self.device:
            raise ValueError(f"rope: the plan must be one of rotary() for head_dim {D} on {self.device}")
        args, outs = [], []
        for x, y in ((q, q_out), (k, k_out)):
            if x is None:
                if y is not None:
                    raise ValueError("rope: an output without its input")
                args += (None, 0, 0, None, 0, 0, 0)
                outs.append(None)
                continue
            if y is None:
                y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            xs, ys, shape = x.stride(), y.stride(), x.shape
            if x.dtype != dt or y.dtype != dt:
                raise ValueError(f"rope: rows must be {dt}")
            if len(shape) != 3 or shape[0] != rows or shape[2] != D or shape != y.shape or xs[2] != 1 or ys[2] != 1:
                raise ValueError(f"rope: rows must be [{rows}, heads, {D}] with contiguous channels, outputs of their inputs' "
                                 "shapes")
            px, py = x.data_ptr(), y.data_ptr()
            if (rows > 1 and (ys[0] == 0 or (px == py and xs[0] != ys[0]))) or (
                    shape[1] > 1 and (ys[1] == 0 or (px == py and xs[1] != ys[1]))):
                raise ValueError("rope: an output must be its input with the same strides or lie apart from it, and have no "
                                 "expanded dimension")
            args += (px, xs[0], xs[1], py, ys[0], ys[1], shape[1])
            outs.append(y)
        self._run("kush_sm100_rope", D, self.cfg.dtype_code, rotary.rotary_dim, int(rotary.interleaved), *args,
                  positions.data_ptr(), int(wide), rotary.turns.data_ptr(), rotary.factor, rows)
        return outs[0], outs[1]

    # ---------------------------------------------------------------- decode
    def splits(self, num_seqs: int, num_kv_heads: int, max_full_pages: int, *, window: int | None = None,
               sinks: int = 0) -> int:
        """Split-KV factor for this device (split_factor); under a window, of the pages a query sees."""
        if window is None:
            return split_factor(num_seqs, num_kv_heads, max_full_pages, self.sms)
        tokens = min(max_full_pages * self.P, window + self.P + sinks)
        if not self._tensor_cores:
            # CUDA cores: a block per tile of 32 q heads, as many on an SM as its shared memory (30, 55 or 104 KB) admits; small
            # splits pay, as a block is bound by its own tiles.  One sequence x 8 kv heads under 8192 tokens: 16 to 32 splits by
            # the tensor cores' rule, 37 or 51 by this one: fp32 of 128 channels 128 -> 108 us, of 64
            # 185 -> 89, 40 heads a kv head 224 -> 138; 4 x 8 of 4096 tokens 189 -> 140, 194 -> 101, 277 -> 250
            units = max(1, num_seqs * num_kv_heads * -(-self.G // 32))
            resident = {64: 7, 128: 4, 256: 2}[self.D]
            return max(1, min(MAX_SPLITS, resident * self.sms // units, tokens // MIN_SIMT_SPLIT))
        # a windowed unit has few pages, so a second wave of CTAs costs as much as the first: count the CTAs that are resident
        # at once.  int8 pages of 32: 3 at head_dim 128 (61 sequences x 4 kv heads of 34 pages: one split 37 us, two 47), 1 at
        # 256 (30 x 4 of 32 pages: one 39 us, two 50).  head_dim 64 with more than 8 heads has 4; counting two measured better
        # (4 x 8 of 4096 tokens: 9 splits 25.8 us, 10 27.6; 61 x 4 of 1000: one 29.4, two 31.8)
        large = self.bits == 8 and self.P == 32
        resident = (1 if large else 2) if self.D == 256 else 2 if self.G > 8 else 3 if large and self.D == 128 else 4
        return split_factor(num_seqs, num_kv_heads, min(max_full_pages, -(-window // self.P) + 1 + -(-sinks // self.P)), self.sms,
                            resident)

    @functools.cached_property
    def _tensor_cores(self) -> bool:
        """Whether the decode of this configuration runs on the tensor cores."""
        return bool(_cuda.decode_tensor_cores(self.cfg))

    def work_size(self, num_seqs: int, num_kv_heads: int, n_splits: int, fused: bool = False) -> int:
        """fp32 elements of the split-KV work buffer: S * Hkv * n_splits * G * (D + 2), the (M, L) pairs first, then
        the unnormalised outputs (the sizing rule of kushkash/_ops.py:195).  fused: S * Hkv more 32-bit slots at the
        end, the counters of decode(fused=True) (they must be 0 before the first fused decode: allocate the buffer
        with torch.zeros; every fused decode leaves them 0)."""
        return num_seqs * num_kv_heads * (n_splits * self.G * (self.D + 2) + (1 if fused else 0))

    def _parts(self, S: int, H: int, n_splits: int, work: torch.Tensor | None,
               fused: bool = False) -> tuple[int, int]:
        n_ml = S * H * n_splits * self.G * 2
        _need(work is not None and work.dtype == torch.float32 and work.is_contiguous()
              and work.numel() >= self.work_size(S, H, n_splits, fused),
              f"decode: n_splits={n_splits} needs a contiguous fp32 work buffer of >= "
              f"{self.work_size(S, H, n_splits, fused)} elements")
        return work.data_ptr(), work.data_ptr() + 4 * n_ml

    def decode(self, q: torch.Tensor, out: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
               seq_lens: torch.Tensor, tail_idx: torch.Tensor, tail_k: torch.Tensor, scale: float, n_splits: int = 1,
               work: torch.Tensor | None = None, *, rotate: bool = False, order: torch.Tensor | None = None,
               fused: bool = False, window: int | None = None, sinks: int = 0) -> None:
        """out[s] = softmax-scaled attention of q[s] over the seq_lens[s] cached tokens of sequence s.  n_splits > 1
        splits each sequence's pages over CTAs (split-KV) and merges them with a second launch; it needs `work`
        (work_size() fp32 elements).  fused: the merge runs inside the decode launch instead (the last CTA of each
        (sequence, kv head) merges; the same output bit for bit); `work` then needs work_size(..., fused=True)
        elements whose last S * Hkv start at 0.  rotate: the cache holds rotated K / V; q is rotated inside the
        kernel and the output rotated back before its store.  order: a contiguous int32 permutation of the
        sequences, CTA x then decoding sequence order[x] (longest_first()); the outputs do not depend on it.
        window: the query sees the last `window` tokens (its own among them) and the first `sinks`; pages without a
        visible token are not read, nor their block-table entries (give splits() the same window and sinks).  Under a
        window the arguments are checked: q and out contiguous [S, H * G, D], int32 index tensors of at least S rows."""
        if window is not None or sinks:
            self._decode_window(q, out, cache, block_table, seq_lens, tail_idx, tail_k, scale, n_splits, work, rotate, order,
                                fused, window, sinks)
            return
        S, H = q.shape[0], tail_k.shape[1]
        ml = o = 0
        if n_splits > 1:
            ml, o = self._parts(S, H, n_splits, work, fused)
        if fused and n_splits > 1:
            if order is not None:
                _need(order.dtype == torch.int32 and order.numel() == S and order.is_contiguous(),
                      "decode: order must be a contiguous int32 permutation of the sequences")
            counters = ml + 4 * S * H * n_splits * self.G * (self.D + 2)
            self._run("kush_sm100_decode_fused_combine", *self._fmt, self.G, q.data_ptr(), out.data_ptr(),
                      *_pool(cache), tail_k.data_ptr(), tail_idx.data_ptr(), block_table.data_ptr(),
                      seq_lens.data_ptr(), block_table.stride(0), H, float(scale), n_splits, ml, o, counters, S,
                      1 if rotate else 0, order.data_ptr() if order is not None else None)
            return
        self._decode(q, out.data_ptr(), cache, block_table, seq_lens, tail_idx, tail_k, scale, n_splits, ml, o,
                     rotate, order)
        if n_splits > 1:
            entry = "kush_sm100_combine_rotated" if rotate else "kush_sm100_combine"
            self._run(entry, self.D, self.cfg.dtype_code, self.G, out.data_ptr(), ml, o, n_splits, H, S)

    def decode_partials(self, q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                        seq_lens: torch.Tensor, tail_idx: torch.Tensor, tail_k: torch.Tensor, scale: float,
                        n_splits: int, work: torch.Tensor) -> tuple[int, int]:
        """The split-KV decode (n_splits >= 2) without its combine: the per-split (M, L) and unnormalised outputs
        in `work`, for a combine that writes elsewhere (the peer gather of KV-head sharding, shard.PeerGather).
        Returns their device addresses (part_ml, part_o)."""
        _need(n_splits >= 2, "decode_partials needs n_splits >= 2")
        S, H = q.shape[0], tail_k.shape[1]
        ml, o = self._parts(S, H, n_splits, work)
        self._decode(q, o, cache, block_table, seq_lens, tail_idx, tail_k, scale, n_splits, ml, o)
        return ml, o

    def _decode(self, q, out_ptr: int, cache, block_table, seq_lens, tail_idx, tail_k, scale: float, n_splits: int,
                part_ml: int, part_o: int, rotate: bool = False, order: torch.Tensor | None = None) -> None:
        S, H = q.shape[0], tail_k.shape[1]
        head = (*self._fmt, self.G, q.data_ptr(), out_ptr, *_pool(cache), tail_k.data_ptr(), tail_idx.data_ptr(),
                block_table.data_ptr(), seq_lens.data_ptr(), block_table.stride(0), H, float(scale), n_splits,
                part_ml or None, part_o or None, S)
        if order is None:
            self._run("kush_sm100_decode_rotated" if rotate else "kush_sm100_decode", *head)
            return
        _need(order.dtype == torch.int32 and order.numel() == S and order.is_contiguous(),
              "decode: order must be a contiguous int32 permutation of the sequences")
        self._run("kush_sm100_decode_ex", *head, 1 if rotate else 0, order.data_ptr())

    def _decode_window(self, q, out, cache, block_table, seq_lens, tail_idx, tail_k, scale: float, n_splits: int,
                       work: torch.Tensor | None, rotate: bool, order: torch.Tensor | None, fused: bool, window: int | None,
                       sinks: int) -> None:
        D, dt, i32, shape, tail = self.D, self.dtype, torch.int32, q.shape, tail_k.shape
        self._here("decode", q, out, cache, block_table, seq_lens, tail_idx, tail_k,
                   *(t for t in (work, order) if t is not None))
        if window is None or window < 1 or sinks < 0:
            raise ValueError(f"decode: window must be >= 1 and sinks >= 0 (sinks need a window), got {window} and {sinks}")
        if not (q.dtype == out.dtype == tail_k.dtype == dt):
            raise ValueError(f"decode: q, out and tail_k must be {dt}")
        if len(tail) != 4 or tail[2] != self.P or tail[3] != D or not tail_k.is_contiguous():
            raise ValueError(f"decode: tail_k must be contiguous [slots, H, {self.P}, {D}]")
        S, H = shape[0], tail[1]
        if len(shape) != 3 or shape[1] != H * self.G or shape[2] != D or out.shape != shape or not (
                q.is_contiguous() and out.is_contiguous()):
            raise ValueError(f"decode: q and out must be contiguous [S, {H * self.G}, {D}] (a part of q|k|v rows: its .contiguous())")
        if (not (seq_lens.dtype == tail_idx.dtype == block_table.dtype == i32)
                or seq_lens.dim() != 1 or tail_idx.dim() != 1 or block_table.dim() != 2
                or min(seq_lens.shape[0], tail_idx.shape[0], block_table.shape[0]) < S
                or not seq_lens.is_contiguous() or not tail_idx.is_contiguous() or block_table.stride(1) != 1):
            raise ValueError("decode: seq_lens and tail_idx must be contiguous int32 [S], block_table [S, pages] int32 with "
                             "contiguous rows")
        if cache.dim() < 2 or cache.shape[1] < H:
            raise ValueError(f"decode: cache must hold the records of {H} kv heads, got {tuple(cache.shape)}")
        part_ml = part_o = counters = address = None
        if n_splits > 1:
            part_ml, part_o = self._parts(S, H, n_splits, work, fused)
            counters = part_ml + 4 * S * H * n_splits * self.G * (D + 2) if fused else None
        if order is not None:
            _need(order.dtype == i32 and order.numel() == S and order.is_contiguous(),
                  "decode: order must be a contiguous int32 permutation of the sequences")
            address = order.data_ptr()
        self._run("kush_sm100_decode_window", *self._fmt, self.G, q.data_ptr(), out.data_ptr(), *_pool(cache),
                  tail_k.data_ptr(), tail_idx.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), block_table.stride(0),
                  H, float(scale), n_splits, part_ml, part_o, counters, S, 1 if rotate else 0, address,
                  min(window, _I32_MAX), min(sinks, _I32_MAX))

    # ---------------------------------------------------------------- chunk attention
    def chunk_splits(self, num_rows: int, num_seqs: int, num_kv_heads: int, max_len: int, *, window: int | None = None,
                     sinks: int = 0) -> int:
        """Split factor of attend_chunk() for this device: row tiles and kv heads that leave SMs free split their keys
        (chunk_split_factor).  num_rows: the step's new rows; max_len: the longest sequence, new rows counted."""
        if window is not None:
            max_len = min(max_len, window + sinks + -(-num_rows // max(1, num_seqs)))
        if self.D != 256 and self.dtype != torch.float32:
            return chunk_split_factor(num_rows, num_seqs, num_kv_heads, self.G, max_len, self.sms)
        # CUDA cores: a block per 32 query rows, as many on an SM as its shared memory (30, 55 or 104 KB) admits.  Few blocks are
        # split until they fill the SMs once, down to 48 tokens; many, whose waves are uneven, four times, in parts that pay for
        # their merge.  By the tensor cores' rule and by this one, 8 kv heads of 4 q heads: a token over 8000 fp32 196 and 97 us,
        # bf16 of 256 channels 282 and 157; 16 x 5 rows over 4000 fp32 of 128 channels 1559 and 558, of 64 1410 and 417, bf16 of 256
        # 2274 and 1092; 300 rows over 4000 1196 and 1115, 857 and 681, 2723 and 2733
        units = max(1, max(num_seqs, -(-num_rows * self.G // 32)) * num_kv_heads)
        blocks = {64: 7, 128: 4, 256: 2}[self.D] * self.sms
        if blocks // units >= 8:
            return max(1, min(MAX_SPLITS, blocks // units, max_len // MIN_SIMT_CHUNK_SPLIT))
        return max(1, min(MAX_SPLITS, 4 * blocks // units, max_len // MIN_CHUNK_SPLIT))

    def chunk_work_size(self, num_rows: int, num_kv_heads: int, n_splits: int) -> int:
        """fp32 elements of attend_chunk()'s work buffer for n_splits > 1: the unnormalised outputs of every row and
        split, then their (M, L) pairs."""
        return num_rows * num_kv_heads * n_splits * self.G * (self.D + 2)

    def attend_chunk(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                     query_start_loc: torch.Tensor, seq_lens: torch.Tensor, tail_idx: torch.Tensor, cache: torch.Tensor,
                     block_table: torch.Tensor, tail_k: torch.Tensor, scale: float, n_splits: int = 1,
                     work: torch.Tensor | None = None, *, window: int | None = None, sinks: int = 0) -> None:
        """Causal attention of a step's new rows over the cached history and themselves, read from the packed records
        (no unpacked copy); call it before write() stores the rows.  Sequence s owns rows [qsl[s], qsl[s+1]) of q
        [rows, H * G, D], k and v [rows, H, D] (row strides free, head stride D) and out [rows, H * G, D]
        (contiguous); seq_lens[s] counts them, as in write().  Any mix of chunk lengths, one token and no history
        included; rows before qsl[0] and from qsl[S] on are left alone.  window, sinks: as in decode(), for every row from its own
        position.  n_splits > 1 (chunk_splits()) divides each tile's keys over more blocks and needs `work`
        (chunk_work_size() fp32 elements).  Over a rotated cache, give it fwht() of q, k and v (write() wants the
        latter two as well) and take fwht() of out."""
        D, G, dt, S = self.D, self.G, self.dtype, seq_lens.shape[0]
        qs, ks, vs, shape = q.stride(), k.stride(), v.stride(), k.shape
        self._here("attend_chunk", q, k, v, out, query_start_loc, seq_lens, tail_idx, cache, block_table, tail_k)
        if not (q.dtype == k.dtype == v.dtype == out.dtype == tail_k.dtype == dt):
            raise ValueError(f"attend_chunk: q, k, v, out and tail_k must be {dt}")
        if len(shape) != 3 or shape[2] != D or v.shape != shape or ks[1:] != (D, 1) or vs[1:] != (D, 1):
            raise ValueError(f"attend_chunk: k and v must be [rows, H, {D}] with head stride {D}")
        rows, H = shape[0], shape[1]
        if tuple(q.shape) != (rows, H * G, D) or qs[1:] != (D, 1):
            raise ValueError(f"attend_chunk: q must be [{rows}, {H * G}, {D}] with head stride {D}")
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError("attend_chunk: out must be contiguous, of q's shape")
        if tuple(tail_k.shape[1:]) != (H, self.P, D) or not tail_k.is_contiguous():
            raise ValueError(f"attend_chunk: tail_k must be contiguous [slots, {H}, {self.P}, {D}]")
        if cache.dim() < 2 or cache.shape[1] < H:
            raise ValueError(f"attend_chunk: cache must hold the records of {H} kv heads, got {tuple(cache.shape)}")
        i32 = torch.int32
        if (not (query_start_loc.dtype == seq_lens.dtype == tail_idx.dtype == block_table.dtype == i32)
                or tuple(query_start_loc.shape) != (S + 1,) or seq_lens.dim() != 1 or tail_idx.dim() != 1 or block_table.dim() != 2
                or tail_idx.shape[0] < S or block_table.shape[0] < S
                or not query_start_loc.is_contiguous() or not seq_lens.is_contiguous() or not tail_idx.is_contiguous()
                or block_table.stride(1) != 1):
            raise ValueError("attend_chunk: query_start_loc [S + 1], seq_lens and tail_idx [S] must be contiguous int32, "
                             "block_table [S, pages] int32 with contiguous rows")
        if (window is None and sinks) or sinks < 0 or (window is not None and window < 1):
            raise ValueError(f"attend_chunk: window must be >= 1 and sinks >= 0 (sinks need a window), got {window} and {sinks}")
        part_o = part_ml = None
        if n_splits > 1:
            need = self.chunk_work_size(rows, H, n_splits)
            _need(work is not None and work.dtype == torch.float32 and work.is_contiguous() and work.numel() >= need
                  and work.get_device() == self.dev, f"attend_chunk: n_splits={n_splits} needs a contiguous fp32 work buffer of >= {need} elements")
            part_o = work.data_ptr()
            part_ml = part_o + 4 * rows * H * n_splits * self.G * D
        self._run("kush_sm100_attend_chunk", *self._fmt, G, q.data_ptr(), qs[0], k.data_ptr(), v.data_ptr(),
                  ks[0], vs[0], out.data_ptr(), query_start_loc.data_ptr(), seq_lens.data_ptr(),
                  tail_idx.data_ptr(), *_pool(cache), tail_k.data_ptr(), *_table(block_table), H, float(scale),
                  min(window, _I32_MAX) if window is not None else 0, min(sinks, _I32_MAX), n_splits, part_ml, part_o, rows,
                  S)

    def longest_first(self, seq_lens: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """A launch order for decode(order=): the sequences by full pages, most first (one small kernel; compute it
        once per step, as the layers share seq_lens)."""
        S = seq_lens.numel()
        _need(seq_lens.dtype == torch.int32 and seq_lens.is_contiguous(), "longest_first: seq_lens must be "
              "contiguous int32")
        order = torch.empty(S, dtype=torch.int32, device=seq_lens.device) if out is None else out
        _need(order.dtype == torch.int32 and order.numel() == S and order.is_contiguous(),
              "longest_first: out must be a contiguous int32 tensor of n_seqs entries")
        self._run("kush_sm100_order_longest_first", seq_lens.data_ptr(), S, self.P, order.data_ptr())
        return order

"""The refusals of the rotary, windowed decode and chunk entry points, and their host-side rules, without a GPU."""
import ctypes
import math

import pytest

P16 = ctypes.c_void_p(16)


def refused(fn, *args):
    from kushkash_b200._cuda import KUSH_ERR_ARG, KUSH_ERR_UNSUPPORTED, last_error, lib
    rc = getattr(lib(), fn)(*args)
    assert rc in (KUSH_ERR_ARG, KUSH_ERR_UNSUPPORTED) and last_error(), (rc, last_error())
    return last_error()


def rope_args(**kw):
    a = dict(head_dim=128, dtype=1, rotary_dim=128, interleaved=0, q=P16, qr=128, qh=128, qo=P16, qor=128, qoh=128, hq=1,
             k=None, kr=0, kh=0, ko=None, kor=0, koh=0, hk=0, positions=P16, pos64=1, turns=P16, factor=1.0, rows=1)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(dtype=3), dict(rotary_dim=3), dict(rotary_dim=130), dict(rotary_dim=0), dict(rows=-1),
                                dict(q=None), dict(qo=None), dict(hk=2), dict(positions=None), dict(turns=None), dict(hq=-1)])
def test_rope_refusals(kw):
    refused("kush_sm100_rope", *rope_args(**kw))


def test_rope_nothing_to_do():
    from kushkash_b200._cuda import lib
    assert lib().kush_sm100_rope(*rope_args(rows=0)) == 0
    assert lib().kush_sm100_rope(*rope_args(hq=0)) == 0


def chunk_args(**kw):
    a = dict(head_dim=128, bits=4, page=16, dtype=1, group=4, q=P16, qs=512, k=P16, v=P16, ks=128, vs=128, out=P16, qsl=P16,
             seq_lens=P16, tail_idx=P16, cache=P16, bs=2624, hs=2624, tail_k=P16, table=P16, max_pages=4, hkv=1, scale=0.1,
             window=0, sinks=0, n_splits=1, ml=None, o=None, rows=4, seqs=1)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(bits=5), dict(page=64), dict(dtype=3), dict(group=0), dict(hkv=0), dict(rows=-1),
                                dict(seqs=-1), dict(window=-1), dict(sinks=-1), dict(n_splits=0), dict(n_splits=2), dict(q=None),
                                dict(k=None), dict(out=None), dict(tail_k=None), dict(qsl=None), dict(cache=ctypes.c_void_p(24)),
                                dict(bs=2625), dict(qs=513), dict(ks=130), dict(q=ctypes.c_void_p(18)),
                                dict(rows=2 ** 31, group=1), dict(n_splits=2, ml=P16, o=ctypes.c_void_p(8))])
def test_chunk_refusals(kw):
    refused("kush_sm100_attend_chunk", *chunk_args(**kw))


def test_chunk_nothing_to_do():
    from kushkash_b200._cuda import lib
    assert lib().kush_sm100_attend_chunk(*chunk_args(rows=0)) == 0
    assert lib().kush_sm100_attend_chunk(*chunk_args(seqs=0)) == 0


def window_args(**kw):
    a = dict(head_dim=128, bits=4, page=16, dtype=1, group=4, q=P16, out=P16, cache=P16, bs=2624, hs=2624, tail_k=P16, tail_idx=P16,
             table=P16, seq_lens=P16, max_pages=4, hkv=1, scale=0.1, n_splits=1, ml=None, o=None, counters=None, seqs=1, flags=0,
             order=None, window=8, sinks=0)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-1), dict(sinks=-1), dict(flags=2), dict(n_splits=2), dict(q=None),
                                dict(head_dim=96), dict(hkv=0)])
def test_window_refusals(kw):
    refused("kush_sm100_decode_window", *window_args(**kw))


def test_rotary_frequencies():
    from kushkash_b200 import rotary_frequencies
    base, one = rotary_frequencies(8, 10000.0)
    assert one == 1.0 and base == pytest.approx([1.0, 0.1, 0.01, 0.001])
    assert rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 2})[0] == pytest.approx([0.5, 0.05, 0.005, 0.0005])
    ntk = rotary_frequencies(8, 10000.0, {"rope_type": "ntk", "factor": 4.0})[0]
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(0.001 / 4)
    yarn, scale = rotary_frequencies(64, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096})
    plain = rotary_frequencies(64)[0]
    assert scale == pytest.approx(0.1 * math.log(4) + 1) and yarn[0] == 1.0 and yarn[-1] == pytest.approx(plain[-1] / 4)
    assert all(p / 4 <= y <= p for y, p in zip(yarn, plain))
    band, one = rotary_frequencies(64, 10000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                                 "high_freq_factor": 4.0, "original_max_position_embeddings": 8192})
    assert one == 1.0 and band[0] == 1.0 and band[-1] == pytest.approx(plain[-1] / 8)
    assert rotary_frequencies(8, 10000.0, {"rope_type": "default"}) == (base, 1.0)
    for bad in ({"rope_type": "linear"}, {"rope_type": "spiral", "factor": 2}, {"rope_type": "yarn", "factor": 2},
                {"rope_type": "linear", "factor": 0}, {"factor": 2.0}):
        with pytest.raises(ValueError):
            rotary_frequencies(8, 10000.0, bad)


def test_chunk_split_factor():
    from kushkash_b200 import chunk_split_factor
    assert chunk_split_factor(2048, 1, 8, 4, 32000, 148) == 1                  # 32 tiles x 8 heads fill the SMs
    assert chunk_split_factor(17, 1, 8, 4, 517, 148) == 2                      # bounded by the tokens
    assert chunk_split_factor(5, 1, 8, 4, 100000, 148) == 18
    assert chunk_split_factor(320, 64, 8, 4, 8192, 148) == 1
    assert chunk_split_factor(1, 1, 1, 1, 1, 148) == 1
    assert chunk_split_factor(0, 0, 1, 1, 0, 148) == 1

"""The 8-bit cache's oracle against closed forms, and the entry points' refusals (no GPU needed)."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import kv_int8 as o_kv


@pytest.mark.parametrize("amax,scale", [
    (127.0, 1.0), (127.5, 2.0), (128.0, 2.0), (63.5, 0.5), (64.0, 1.0), (1.0, 2.0**-6), (0.0, 2.0**-126),
    (2.0**-130, 2.0**-126), (3.3895313892515355e38, 2.0**122), (1.984375, 2.0**-6), (1.9921875, 2.0**-5),
])
def test_scale_is_the_least_power_of_two(amax, scale):
    assert o_kv.scale_for(amax) == scale
    assert amax <= 127 * scale and (scale == 2.0**-126 or amax > 127 * scale / 2)


def _empty(pages=2, ps=16, heads=1, d=4):
    return (np.full((pages, 2, ps, heads, d), 99, np.int8), np.full((pages, 2, ps // 16, heads), 7.0, np.float32))


def test_growth_rescales_what_the_block_holds():
    codes, scales = _empty()
    k = np.array([[[100.0, -50.0, 3.0, 1.0]]])
    o_kv.write(codes, scales, k, k / 2, [1], [0])
    assert scales[1, 0, 0, 0] == 1.0 and scales[1, 1, 0, 0] == 0.5
    assert codes[1, 0, 0, 0].tolist() == [100, -50, 3, 1] == codes[1, 1, 0, 0].tolist()
    o_kv.write(codes, scales, 4 * k, k / 4, [1], [1])  # K grows by 4, V does not
    assert scales[1, 0, 0, 0] == 4.0 and scales[1, 1, 0, 0] == 0.5
    assert codes[1, 0, 0, 0].tolist() == [25, -12, 1, 0]  # 12.5 -> 12, 0.75 -> 1, 0.25 -> 0
    assert codes[1, 0, 1, 0].tolist() == [100, -50, 3, 1]
    assert (codes[1, 0, 2:] == 99).all() and (codes[0] == 99).all() and (scales[0] == 7.0).all()


def test_error_stays_below_one_step():
    """However often a block grows: half a step of each scale, and the scales double at least."""

    rng = np.random.default_rng(3)
    for _ in range(20):
        codes, scales = _empty(pages=1, heads=1, d=8)
        x = rng.standard_normal((16, 1, 8)) * 2.0 ** rng.uniform(-2, 5, (16, 1, 1)).cumsum(0)
        for t in range(16):
            o_kv.write(codes, scales, x[t : t + 1], x[t : t + 1], [0], [t])
        got = o_kv.values(codes, scales)[0, 0]
        assert (np.abs(got - x) < scales[0, 0, 0, 0]).all()
        assert scales[0, 0, 0, 0] == o_kv.scale_for(np.abs(x).max())


def test_attention_closed_forms():
    codes, scales = _empty(pages=3, heads=1, d=4)
    scales[:] = 0.25
    rng = np.random.default_rng(1)
    codes[:] = rng.integers(-127, 128, codes.shape)
    q = rng.standard_normal((2, 2, 4))
    out, bound = o_kv.attention(q, codes, scales, [0, 1, 1], [2], [1, 1])
    assert np.array_equal(out[0], np.broadcast_to(codes[2, 1, 0, 0] * 0.25, (2, 4)))  # one key: its V
    assert (out[1] == 0).all() and (bound[1] == 0).all()  # no page
    codes[:, 0] = 5  # equal keys: the mean of V
    out, bound = o_kv.attention(q[:1], codes, scales, [0, 2], [2, 0], [3])
    v = np.concatenate((codes[2, 1, :, 0], codes[0, 1, :3, 0])) * 0.25
    assert np.allclose(out[0], v.mean(0), rtol=1e-12) and (bound[0] < 0.03 * np.abs(v).max()).all()


def test_attention_by_rows_is_attention():
    """Rows at once against query by query: values and bounds; and a page outside the pool against the same keys left out."""

    rng = np.random.default_rng(5)
    codes = rng.integers(-127, 128, (9, 2, 16, 2, 8)).astype(np.int8)
    scales = (2.0 ** rng.integers(-8, -4, (9, 2, 1, 2))).astype(np.float32)
    q = rng.standard_normal((24, 4, 8))
    where = ([0, 3, 3, 8], [4, 0, 7, 1, 2, 3, 8, 5], [5, 1, 16], [0, 9, 11, 24])
    for got, want in zip(o_kv.attention_rows(q, codes, scales, *where), o_kv.attention(q, codes, scales, *where)):
        assert np.allclose(got, want, rtol=1e-9, atol=1e-300)
    assert (o_kv.attention_rows(q, codes, scales, *where)[0][9:11] == 0).all()
    out, bound = o_kv.attention_rows(q[:1], codes, scales, [0, 3], [4, 9, 2], [16], [0, 1])
    want, wide = o_kv.attention(q[:1], codes, scales, [0, 2], [4, 2], [16], [0, 1])
    assert np.allclose(out, want, rtol=1e-12) and np.allclose(bound, wide, rtol=1e-9)


# -- refusals ------------------------------------------------------------------------------------------


def _args(tokens=3, pages=4, ps=16, heads=2, d=64):
    return SimpleNamespace(
        key=torch.zeros(tokens, heads, d, dtype=torch.bfloat16), value=torch.zeros(tokens, heads, d, dtype=torch.bfloat16),
        layer_cache=torch.zeros(pages, 2, ps, heads, d, dtype=torch.int8),
        layer_scales=torch.zeros(pages, 2, max(ps // 16, 1), heads),
        write_pages=torch.zeros(tokens, dtype=torch.long), write_offsets=torch.arange(tokens))


@pytest.mark.parametrize("name,bad,error", [
    ("key", lambda t: t.float(), TypeError),
    ("value", lambda t: t.half(), TypeError),
    ("key", lambda t: t[:2], ValueError),
    ("key", lambda t: t[:, :1], ValueError),
    ("value", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), ValueError),
    ("layer_cache", lambda t: t.view(torch.uint8), TypeError),
    ("layer_cache", lambda t: t[:, :1], ValueError),
    ("layer_cache", lambda t: t[0], ValueError),
    ("layer_cache", lambda t: t[:, :, :8], TypeError),
    ("layer_cache", lambda t: t.repeat(1, 1, 3, 1, 1), TypeError),
    ("layer_scales", lambda t: t.double(), TypeError),
    ("layer_scales", lambda t: t[:3], ValueError),
    ("write_pages", lambda t: t.int(), TypeError),
    ("write_pages", lambda t: t[:2], ValueError),
    ("write_offsets", lambda t: torch.arange(6)[::2], ValueError),
    (None, None, ValueError),  # the call itself, but on the CPU
])
def test_write_refusals(nq, name, bad, error):
    from nari_qwen3_tts_amd import kernels

    args = _args()
    if name:
        setattr(args, name, bad(getattr(args, name)))
    with pytest.raises(error):
        kernels.paged_cache_write_int8_(**vars(args))


def _metadata(rows=2, **other):
    fields = dict(qo_indptr=torch.arange(rows + 1, dtype=torch.int32),
                  paged_kv_indptr=torch.arange(rows + 1, dtype=torch.int32),
                  paged_kv_indices=torch.arange(rows, dtype=torch.int32),
                  paged_kv_last_page_len=torch.ones(rows, dtype=torch.int32))
    fields.update(other)
    return SimpleNamespace(**fields)


@pytest.mark.parametrize("change,error", [
    (dict(query=torch.zeros(2, 4, 64)), TypeError),
    (dict(query=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), ValueError),
    (dict(query=torch.zeros(2, 4, 128, dtype=torch.bfloat16)), ValueError),
    (dict(query=torch.zeros(4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(out=torch.zeros(2, 4, 64)), TypeError),
    (dict(out=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(metadata=_metadata(paged_kv_indptr=torch.arange(3))), TypeError),
    (dict(metadata=_metadata(qo_indptr=torch.arange(4, dtype=torch.int32))), ValueError),
    (dict(metadata=_metadata(paged_kv_last_page_len=torch.ones(1, dtype=torch.int32))), ValueError),
    (dict(metadata=_metadata(paged_kv_indices=torch.arange(4, dtype=torch.int32)[::2])), ValueError),
    (dict(metadata=_metadata(qo_indptr=None), parts=3), ValueError),
    (dict(metadata=_metadata(rows=3, qo_indptr=None)), ValueError),
    (dict(), ValueError),  # the call itself, but on the CPU
])
def test_attention_refusals(nq, change, error):
    from nari_qwen3_tts_amd import kernels

    a = _args()
    args = dict(query=torch.zeros(2, 4, 64, dtype=torch.bfloat16), layer_cache=a.layer_cache,
                layer_scales=a.layer_scales, metadata=_metadata())
    args.update(change)
    with pytest.raises(error):
        kernels.paged_attention_int8(**args)


def test_host_checks_of_the_c_entries(nq):
    """Refused before any launch (placeholder pointers)."""

    from nari_qwen3_tts_amd import _lib

    lib = _lib.load()

    def write(key=16, k_s0=128, tokens=2, heads=2, d=64, codes=16, c_slot=128, pages=4, ps=16):
        return lib.nq_kv_int8_write(key, k_s0, 64, 16, 128, 64, tokens, heads, d, codes, 4096, 2048, c_slot, 64, 16, 4,
                                    2, 2, 1, pages, ps, 16, 16, None, None)

    assert write(tokens=0) == 0
    assert write(tokens=-1) == -1 and write(heads=0) == -1 and write(codes=None) == -1 and write(pages=0) == -1
    assert write(ps=24) == -1 and write(ps=8) == -2 and write(d=96) == -2
    assert write(key=8) == -2 and write(k_s0=100) == -2 and write(codes=8) == -2 and write(c_slot=120) == -2

    size = lib.nq_paged_attention_int8_workspace_bytes
    assert size(4, 2, 16, 8, 128, 3) > 0
    for bad in ((0, 2, 16, 8, 128, 3), (4, 0, 16, 8, 128, 3), (4, 2, 15, 8, 128, 3), (4, 2, 17, 1, 128, 3),
                (4, 2, 16, 8, 96, 3), (4, 2, 16, 8, 128, 0), (4, 2, 16, 8, 128, 4), (4, 2, 4, 8, 128, 1)):
        assert size(*bad) == -1, bad

    def attend(qo=16, parts=3, q=16, q_s0=1024, ws=16, ws_bytes=1 << 40, hq=16, n=2, ids=2, ps=16, tokens=4):
        return lib.nq_paged_attention_int8(qo, 16, 16, 16, n, ids, q, q_s0, 64, tokens, 16, 32768, 16384, 1024, 128, 16,
                                           16, 8, 8, 1, 4, ps, hq, 8, 128, 0.1, 16, 2048, 128, parts, ws, ws_bytes,
                                           None, None)

    assert attend(n=0) == 0 and attend(tokens=0) == 0
    assert attend(qo=None) == -1 and attend(parts=0) == -1 and attend(parts=4) == -1 and attend(hq=12) == -1
    assert attend(ws=None) == -1 and attend(ws_bytes=64) == -1 and attend(ws=8) == -1
    assert attend(qo=None, parts=1, n=5) == -1  # more rows than queries
    assert attend(q=8) == -2 and attend(q_s0=1020) == -2 and attend(ps=8) == -2
    assert attend(ids=1 << 28) == -2  # 2^32 slots


def test_sm_scale_that_is_not_finite_is_refused(nq):
    """Also where the factor log2(e) or the entry's fp32 takes it there."""

    from nari_qwen3_tts_amd import _lib, kernels

    a = _args()
    lib = _lib.load()
    for bad in (float("nan"), float("inf"), float("-inf"), 3e38, 1e300):
        with pytest.raises(ValueError, match="sm_scale"):
            kernels.paged_attention_int8(torch.zeros(2, 4, 64, dtype=torch.bfloat16), a.layer_cache, a.layer_scales,
                                         _metadata(), sm_scale=bad)
        assert lib.nq_paged_attention_int8(16, 16, 16, 16, 2, 2, 16, 1024, 64, 4, 16, 32768, 16384, 1024, 128, 16, 16, 8, 8,
                                           1, 4, 16, 16, 8, 128, bad, 16, 2048, 128, 3, 16, 1 << 40, None, None) == -1


def test_page_lists_near_2_31_slots_are_refused(nq):
    """The last key tile of such a row would pass 2^31."""

    from nari_qwen3_tts_amd import _lib

    lib = _lib.load()
    for ids, d in ((0x7FFFFFFF // 16, 128), (0x7FFF0000 // 16 + 1, 64)):
        assert lib.nq_paged_attention_int8(16, 16, 16, 16, 2, ids, 16, 1024, 64, 4, 16, 32768, 16384, 1024, 128, 16, 16, 8,
                                           8, 1, 4, 16, 16, 8, d, 0.1, 16, 2048, 128, 3, 16, 1 << 40, None, None) == -2

"""The paged K/V cache in 8 bits against its float64 oracle: codes and scales equal, attention within the
oracle's derived bound."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import kv_int8 as o_kv

pytestmark = pytest.mark.gpu


def _pool(device, rng, pages, ps, heads, d, fill=True):
    codes = rng.integers(-127, 128, (pages, 2, ps, heads, d)).astype(np.int8)
    scales = (2.0 ** rng.integers(-9, -4, (pages, 2, ps // 16, heads))).astype(np.float32)
    return torch.from_numpy(codes).to(device), torch.from_numpy(scales).to(device)


def _bf16(rng, device, *shape, size=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * size).astype(np.float32)).to(device, torch.bfloat16)


def _slots(device, pages, offsets):
    return (torch.tensor(pages, dtype=torch.long, device=device), torch.tensor(offsets, dtype=torch.long, device=device))


def _check_write(codes, scales, key, value, pages, offsets, status=None):
    from nari_qwen3_tts_amd.kernels import paged_cache_write_int8_

    want_c, want_s = codes.cpu().numpy().copy(), scales.cpu().numpy().copy()
    o_kv.write(want_c, want_s, to_np(key), to_np(value), pages.tolist(), offsets.tolist())
    assert paged_cache_write_int8_(key, value, codes, scales, pages, offsets, status) is None
    assert np.array_equal(scales.cpu().numpy(), want_s, equal_nan=True)
    assert np.array_equal(codes.cpu().numpy(), want_c)


@pytest.mark.parametrize("heads,d,ps", [(8, 128, 16), (1, 64, 64), (3, 128, 32), (8, 64, 16), (2, 128, 256)])
@pytest.mark.parametrize("starts,news", [
    ([0], [1]), ([5], [1]), ([15], [2]), ([16], [16]), ([3], [40]), ([0, 7, 31, 16], [17, 1, 33, 15]),
    (list(range(40)), [1] * 40), ([0, 9], [700, 130]),
])
def test_write(nq, device, heads, d, ps, starts, news):
    """Rows that begin anywhere in a block; the last two lists are past one token a wave and past two waves' tokens."""

    rng = np.random.default_rng(len(starts) * 100 + ps + d)
    each = [-(-(s + n) // ps) for s, n in zip(starts, news)]
    codes, scales = _pool(device, rng, sum(each) + 3, ps, heads, d)
    order, pages, offsets, at = rng.permutation(sum(each) + 3), [], [], 0
    for s, n, k in zip(starts, news, each):
        pages += [order[at + i // ps] for i in range(s, s + n)]
        offsets += [i % ps for i in range(s, s + n)]
        at += k
    size = 2.0 ** rng.uniform(-8, 3, (len(pages), 1, 1))
    key, value = _bf16(rng, device, len(pages), heads, d, size=size), _bf16(rng, device, len(pages), heads, d)
    _check_write(codes, scales, key, value, *_slots(device, pages, offsets))


def test_write_one_token_at_a_time_while_the_range_grows(nq, device):
    rng = np.random.default_rng(11)
    codes, scales = _pool(device, rng, 2, 32, 2, 128)
    for t in range(40):
        x = _bf16(rng, device, 2, 1, 2, 128, size=2.0 ** (0.7 * (t % 16)))
        _check_write(codes, scales, x[0], x[1], *_slots(device, [t // 32], [t % 32]))


def test_write_extremes(nq, device):
    """Zeros, the smallest and largest bf16 values, ties, and a block that holds NaN or an infinity."""

    rng = np.random.default_rng(12)
    codes, scales = _pool(device, rng, 8, 16, 1, 64)
    key = torch.zeros(8, 1, 64, dtype=torch.bfloat16, device=device)
    key[1] = 9.183549615799121e-41  # the smallest bf16
    key[2], key[2, 0, 1] = 3.3895313892515355e38, 1.7e38
    key[3, 0, :4] = torch.tensor([100.0, 50.5, 49.5, -0.5])
    key[4, 0, 3] = float("nan")
    key[5, 0, 3] = float("-inf")
    key[6] = 1e-38
    key[7, 0, :2] = torch.tensor([127.5, 127.0])
    _check_write(codes, scales, key, key.flip(0).contiguous(), *_slots(device, list(range(8)), [0, 1] * 4))
    # a later token does not bring a NaN block back; a write at its start does
    _check_write(codes, scales, key[:2], key[:2], *_slots(device, [4, 4], [2, 3]))
    _check_write(codes, scales, key[:1], key[:1], *_slots(device, [4], [0]))


def test_write_skips_slots_outside_the_pool(nq, device):
    rng = np.random.default_rng(13)
    codes, scales = _pool(device, rng, 3, 16, 2, 64)
    x = _bf16(rng, device, 2, 6, 2, 64)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    _check_write(codes, scales, x[0], x[1], *_slots(device, [0, 0, 2, 2, 1, 1], [3, 4, 0, 1, 9, 10]), status)
    assert int(status) == 0
    _check_write(codes, scales, x[0], x[1], *_slots(device, [0, -1, 2, 3, 1, 1 << 40], [5, 6, 16, 0, -1, 0]), status)
    assert int(status) == -1


def test_write_strided(nq, device):
    """K and V as slices of a packed projection; codes and scales in other orders than the tested ones."""

    rng = np.random.default_rng(14)
    qkv = _bf16(rng, device, 21, 8, 128)
    codes = torch.zeros(4, 2, 3, 16, 128, dtype=torch.int8, device=device).transpose(2, 3)[:, :, :, 1:]
    scales = torch.zeros(2, 2, 1, 4, device=device).permute(3, 0, 2, 1)
    _check_write(codes, scales, qkv[:, 4:6], qkv[:, 6:8], *_slots(device, [2] * 13 + [0] * 8, [*range(3, 16), *range(8)]))
    _check_write(codes, scales, qkv[:0, 4:6], qkv[:0, 6:8], *_slots(device, [], []))


@pytest.mark.parametrize("d,heads,ps,tokens", [(128, 8, 16, 37), (64, 3, 64, 1), (128, 1, 32, 300), (64, 8, 16, 0)])
def test_read(nq, device, d, heads, ps, tokens):
    from nari_qwen3_tts_amd.kernels import paged_cache_read_int8

    rng = np.random.default_rng(15)
    codes, scales = _pool(device, rng, 9, ps, heads, d)
    p, o = rng.integers(0, 9, tokens), rng.integers(0, ps, tokens)
    pages, offsets = _slots(device, p.tolist(), o.tolist())
    want = o_kv.values(codes.cpu().numpy(), scales.cpu().numpy())[p, :, o]
    for out in (None, torch.zeros(tokens, 2 * heads + 1, d, dtype=torch.bfloat16, device=device)):
        k, v = paged_cache_read_int8(codes, scales, pages, offsets, None if out is None else out[:, :heads],
                                     None if out is None else out[:, heads + 1:])
        assert np.array_equal(to_np(k), want[:, 0]) and np.array_equal(to_np(v), want[:, 1])


def test_read_outside_the_pool(nq, device):
    from nari_qwen3_tts_amd.kernels import paged_cache_read_int8

    rng = np.random.default_rng(16)
    codes, scales = _pool(device, rng, 3, 16, 2, 64)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    k, v = paged_cache_read_int8(codes, scales, *_slots(device, [1, 3, -1, 0, 0], [2, 0, 0, 16, -1]), status=status)
    assert int(status) == -1 and not k[1:].any() and not v[1:].any() and k[0].any()


def test_write_over_discarded_tokens(nq, device):
    """A slot written again: the block keeps the step of a discarded outlier, at most one step off, and a discarded NaN, until
    it is written from its first slot."""

    from nari_qwen3_tts_amd.kernels import paged_cache_read_int8

    rng = np.random.default_rng(18)
    codes, scales = _pool(device, rng, 2, 16, 2, 64)
    x = _bf16(rng, device, 2, 8, 2, 64)
    at = _slots(device, [1] * 8, list(range(8)))
    for slots, values in ((slice(0, 5), x[:, :5]), (slice(5, 6), x[:, 5:6] * 64.0), (slice(5, 8), x[:, 5:])):
        _check_write(codes, scales, values[0], values[1], at[0][slots], at[1][slots])
    for got, want, step in zip(paged_cache_read_int8(codes, scales, *at), x, scales[1, :, 0]):
        off = (got.float() - want.float()).abs()
        assert (off < step[:, None]).all() and step.min() >= 0.5  # 64 times values of some 2 in 127 codes
    bad = x[:, 5:6].clone()
    bad[0, 0, 1, 3] = float("nan")
    for values in (bad, x[:, 5:6]):
        _check_write(codes, scales, values[0], values[1], at[0][5:6], at[1][5:6])
        assert scales[1, 0, 0, 1].isnan() and scales[1, 1].isfinite().all()
    _check_write(codes, scales, x[0], x[1], *at)
    assert scales[1].isfinite().all() and (scales[1] <= 2.0**-4).all()


# -- attention -----------------------------------------------------------------------------------------


def _batch(device, seed, kv_lens, q_lens, *, hq, hkv, d, ps, spare=5, tail=0):
    """A ragged batch over a permuted pool; ``tail`` query tokens of no row behind the last."""

    rng = np.random.default_rng(seed)
    pages = [-(-n // ps) for n in kv_lens]
    total = sum(pages) + spare
    codes, scales = _pool(device, rng, total, ps, hkv, d)
    ids = rng.permutation(total)[: sum(pages)]
    indptr = np.concatenate(([0], np.cumsum(pages)))
    last = [(n - 1) % ps + 1 if n else 1 for n in kv_lens]
    tokens = len(kv_lens) if q_lens is None else sum(q_lens)
    q = _bf16(rng, device, tokens + tail, hq, d)

    def int32(x):
        return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)

    meta = SimpleNamespace(
        qo_indptr=None if q_lens is None else int32(np.concatenate(([0], np.cumsum(q_lens)))),
        paged_kv_indptr=int32(indptr), paged_kv_indices=int32(ids), paged_kv_last_page_len=int32(last))
    return q, codes, scales, meta


def _want(q, codes, scales, meta, sm_scale=None):
    m = [None if t is None else t.cpu().numpy() for t in (
        meta.paged_kv_indptr, meta.paged_kv_indices, meta.paged_kv_last_page_len, meta.qo_indptr)]
    return o_kv.attention(to_np(q), codes.cpu().numpy(), scales.cpu().numpy(), *m, sm_scale=sm_scale)


def _compare(out, want, bound, label=""):
    got = to_np(out).astype(np.float64)
    has = ~np.isnan(want)
    excess = np.abs(got - want)[has] - bound[has]
    assert np.isfinite(got[has]).all() and excess.max(initial=-1.0) <= 0, f"{label}: over by {excess.max():.3g}"
    return got


def _check(q, codes, scales, meta, label="", **kwargs):
    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    status = torch.zeros(1, dtype=torch.int32, device=q.device)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=q.device)
    assert paged_attention_int8(q, codes, scales, meta, status=status, out=out, **kwargs) is out
    assert int(status) == 0
    got = _compare(out, *_want(q, codes, scales, meta, kwargs.get("sm_scale")), label)
    again = paged_attention_int8(q, codes, scales, meta, out=torch.full_like(out, 7.0), **kwargs)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16)), label
    return got


DECODE_LENGTHS = [
    [1], [2], [16], [17], [333], [31, 0, 32, 33, 1, 48, 0], [0], [1500, 3, 700], [40] * 9 + [2500] + [5] * 70,
]


@pytest.mark.parametrize("hq,hkv,d,ps", [(16, 8, 128, 16), (16, 8, 64, 16), (8, 8, 128, 32), (16, 2, 128, 64),
                                         (16, 1, 128, 16), (16, 1, 64, 128), (7, 1, 128, 16), (6, 2, 64, 32)])
@pytest.mark.parametrize("case", range(len(DECODE_LENGTHS)))
def test_decode(nq, device, hq, hkv, d, ps, case):
    q, codes, scales, meta = _batch(device, 100 + case, DECODE_LENGTHS[case], None, hq=hq, hkv=hkv, d=d, ps=ps)
    got = _check(q, codes, scales, meta, f"{hq}/{hkv}/{d} page {ps}, lengths {DECODE_LENGTHS[case][:9]}")
    assert all((got[r] == 0).all() for r, n in enumerate(DECODE_LENGTHS[case]) if n == 0)


def test_decode_long(nq, device):
    """Spans of more blocks than one window of 64: 300,000 keys, and rows beside them."""

    q, codes, scales, meta = _batch(device, 120, [9, 300001, 40], None, hq=8, hkv=8, d=64, ps=16)
    _check(q, codes, scales, meta, "long")


PREFILL = [  # (keys, queries) of each row
    ([1], [1]), ([2], [2]), ([64], [64]), ([65], [64]), ([100], [3]), ([33, 0, 70, 5], [33, 2, 1, 5]),
    ([3], [9]),  # more queries than keys: the first six see none
    ([200, 17, 131], [129, 17, 131]), ([700], [70]), ([0, 40, 0], [0, 40, 3]), ([300, 300, 300, 300], [1, 2, 1, 1]),
]


@pytest.mark.parametrize("hq,hkv,d,ps", [(16, 8, 128, 16), (16, 8, 64, 32), (4, 4, 128, 64), (16, 1, 128, 16),
                                         (7, 1, 64, 16), (6, 2, 128, 128)])
@pytest.mark.parametrize("case", range(len(PREFILL)))
def test_prefill(nq, device, hq, hkv, d, ps, case):
    """As one launch for all rows, and with the rows of one query through the decode launch."""

    from nari_qwen3_tts_amd import _lib

    keys, queries = PREFILL[case]
    q, codes, scales, meta = _batch(device, 200 + case, keys, queries, hq=hq, hkv=hkv, d=d, ps=ps, tail=3)
    for parts in (_lib.NQ_ATTN_PREFILL, None):
        got = _check(q, codes, scales, meta, f"{hq}/{hkv}/{d} page {ps}, parts {parts}, {PREFILL[case]}", parts=parts)
        assert (got[sum(queries):] == 7.0).all()  # tokens behind the last row
        at = 0
        for n, m in zip(keys, queries):
            assert (got[at:at + max(0, m - n)] == 0).all()
            at += m


def test_prefill_in_pieces(nq, device):
    """Few tiles over long key ranges: pieces joined by the second launch; the last queries of a row that
    ends inside a page."""

    q, codes, scales, meta = _batch(device, 230, [2100, 901], [20, 13], hq=4, hkv=2, d=128, ps=64)
    _check(q, codes, scales, meta, "pieces")


def test_parts_leave_the_other_rows(nq, device):
    from nari_qwen3_tts_amd import _lib
    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    q, codes, scales, meta = _batch(device, 240, [50, 20, 90], [1, 7, 1], hq=4, hkv=2, d=64, ps=16)
    out = torch.full_like(q, 7.0)
    paged_attention_int8(q, codes, scales, meta, parts=_lib.NQ_ATTN_DECODE, out=out)
    want, bound = _want(q, codes, scales, meta)
    assert (out[1:8] == 7.0).all()
    rows = [0, 8]
    _compare(out[rows], want[rows], bound[rows])


def test_strides_and_scale(nq, device):
    """Queries sliced from a packed projection, a strided output, a head-major cache, another sm_scale."""

    q, codes, scales, meta = _batch(device, 250, [77, 300, 5], [1, 40, 5], hq=8, hkv=2, d=128, ps=32)
    packed = torch.zeros(q.shape[0], 12, 128, dtype=torch.bfloat16, device=device)
    packed[:, 2:10] = q
    out = torch.full((q.shape[0], 3, 8, 128), 7.0, dtype=torch.bfloat16, device=device)
    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    heads_first = codes.transpose(2, 3).contiguous().transpose(2, 3)
    blocks_last = scales.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0)
    paged_attention_int8(packed[:, 2:10], heads_first, blocks_last, meta, sm_scale=0.31, out=out[:, 1])
    _compare(out[:, 1], *_want(q, codes, scales, meta, 0.31))
    assert (out[:, 0] == 7.0).all() and (out[:, 2] == 7.0).all()


def test_what_is_masked_does_not_reach_the_output(nq, device):
    """Codes behind the last key, and whole blocks behind a query's last key whose scale is NaN or infinite,
    within its page and within its tile."""

    from nari_qwen3_tts_amd import _lib
    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    for keys, queries in (([20, 70], None), ([20, 70], [20, 30])):
        q, codes, scales, meta = _batch(device, 260, keys, queries, hq=4, hkv=2, d=128, ps=64)
        want, bound = _want(q, codes, scales, meta)
        ids = meta.paged_kv_indices.cpu().tolist()  # pages of 64: [row 0], [row 1, row 1]
        scales[ids[0], :, 2:] = float("nan")
        scales[ids[2], 0, 1:], scales[ids[2], 1, 1:] = float("inf"), float("nan")
        out = paged_attention_int8(q, codes, scales, meta)
        _compare(out, want, bound)
        if queries:  # keys 64 .. 69, a block of their own, are seen by row 1's last six queries alone
            scales[ids[2]] = float("nan")
            out = paged_attention_int8(q, codes, scales, meta, parts=_lib.NQ_ATTN_PREFILL)
            _compare(out[:44], want[:44], bound[:44])
            assert out[44:].isnan().all()


def test_infinite_and_nan_inputs_answer_nan(nq, device):
    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    q, codes, scales, meta = _batch(device, 270, [40, 40, 40, 40], [1, 2, 1, 2], hq=4, hkv=2, d=64, ps=16)
    q[0, 0, 3] = float("nan")
    q[1, 1, 5] = float("inf")
    want, bound = _want(q, codes, scales, meta)
    out = paged_attention_int8(q, codes, scales, meta)
    assert out[0, 0].isnan().all() and out[1, 1].isnan().all()
    keep = torch.ones(6, 4, dtype=torch.bool)
    keep[0, 0] = keep[1, 1] = False
    _compare(out[keep.to(device)], want[keep.numpy()], bound[keep.numpy()])


def test_pages_outside_the_pool_are_skipped(nq, device):
    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    for queries in (None, [1, 3, 9]):
        q, codes, scales, meta = _batch(device, 280, [48, 16, 41], queries, hq=4, hkv=2, d=128, ps=16)
        meta.paged_kv_indices[1] = codes.shape[0]
        meta.paged_kv_indices[3] = -1  # row 1's only page
        status = torch.zeros(1, dtype=torch.int32, device=device)
        out = paged_attention_int8(q, codes, scales, meta, status=status)
        assert int(status) == -1
        first = 1 if queries is None else 3
        assert not out[1:1 + first].any()
        # row 0 without its middle page: its first and last, one query that sees them all
        ids = meta.paged_kv_indices.cpu().numpy()
        want, bound = o_kv.attention(to_np(q[:1]), codes.cpu().numpy(), scales.cpu().numpy(), [0, 2], ids[[0, 2]], [16])
        _compare(out[:1], want, bound)


def test_offsets_past_32_bits(nq, device):
    """A layer of 5 GB: pages whose codes begin past 2^32 bytes."""

    from nari_qwen3_tts_amd.kernels import paged_attention_int8, paged_cache_read_int8, paged_cache_write_int8_

    pages, ps, heads, d = 160000, 16, 8, 128
    codes = torch.zeros(pages, 2, ps, heads, d, dtype=torch.int8, device=device)
    scales = torch.zeros(pages, 2, 1, heads, device=device)
    rng = np.random.default_rng(290)
    ids = [159999, 3, 140000, 70000]
    slots = [(ids[i // 16], i % 16) for i in range(60)]
    at = _slots(device, [s[0] for s in slots], [s[1] for s in slots])
    x = _bf16(rng, device, 2, 60, heads, d)
    paged_cache_write_int8_(x[0], x[1], codes, scales, *at)
    k, v = paged_cache_read_int8(codes, scales, *at)
    small_c, small_s = codes[ids].cpu().numpy(), scales[ids].cpu().numpy()
    want_c, want_s = np.zeros_like(small_c), np.zeros_like(small_s)
    o_kv.write(want_c, want_s, to_np(x[0]), to_np(x[1]), [i // 16 for i in range(60)], [i % 16 for i in range(60)])
    assert np.array_equal(small_c, want_c) and np.array_equal(small_s, want_s)
    values = o_kv.values(want_c, want_s)
    assert np.array_equal(to_np(k), np.stack([values[i // 16, 0, i % 16] for i in range(60)]))
    for queries in (None, [30]):
        n = 1 if queries is None else 30
        q = _bf16(rng, device, n, 16, d)
        meta = SimpleNamespace(
            qo_indptr=None if queries is None else torch.tensor([0, n], dtype=torch.int32, device=device),
            paged_kv_indptr=torch.tensor([0, 4], dtype=torch.int32, device=device),
            paged_kv_indices=torch.tensor(ids, dtype=torch.int32, device=device),
            paged_kv_last_page_len=torch.tensor([12], dtype=torch.int32, device=device))
        out = paged_attention_int8(q, codes, scales, meta)
        want, bound = o_kv.attention(to_np(q), want_c, want_s, [0, 4], np.arange(4), [12],
                                     None if queries is None else [0, n])
        _compare(out, want, bound)


def test_graph_of_write_and_attention(nq, device):
    """A decode step and a prompt chunk, captured: write, then attend, replayed with other inputs and other
    lengths, eager work in between; the same bits as the eager calls."""

    from nari_qwen3_tts_amd.kernels import paged_attention_int8, paged_cache_write_int8_

    for queries in (None, [1, 19, 1]):
        lens = [30, 19, 300]
        q, codes, scales, meta = _batch(device, 300, lens, queries, hq=16, hkv=8, d=128, ps=16)
        n = q.shape[0]
        rng = np.random.default_rng(301)
        kv = _bf16(rng, device, 2, n, 8, 128)
        ids, indptr = meta.paged_kv_indices.cpu().tolist(), meta.paged_kv_indptr.cpu().tolist()
        pages, offsets = [], []
        for r, m in enumerate(queries or [1, 1, 1]):
            pages += [ids[indptr[r] + i // 16] for i in range(lens[r] - m, lens[r])]
            offsets += [i % 16 for i in range(lens[r] - m, lens[r])]
        at = _slots(device, pages, offsets)
        out = torch.zeros_like(q)

        def step(codes, scales, out):
            paged_cache_write_int8_(kv[0], kv[1], codes, scales, *at)
            paged_attention_int8(q, codes, scales, meta, out=out)

        start = codes.clone(), scales.clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(codes, scales, out)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(codes, scales, out)
        for i in range(4):
            codes.copy_(start[0])
            scales.copy_(start[1])
            q.copy_(_bf16(rng, device, *q.shape))
            kv.copy_(_bf16(rng, device, *kv.shape, size=1.5**i))
            mine = codes.clone(), scales.clone(), torch.zeros_like(out)
            out.fill_(float("nan"))
            graph.replay()
            step(*mine)
            torch.cuda.synchronize()
            assert torch.equal(codes, mine[0]) and torch.equal(scales, mine[1])
            assert torch.equal(out.view(torch.int16), mine[2].view(torch.int16))
            _compare(out, *_want(q, codes, scales, meta))


def test_workspace(nq, device):
    from nari_qwen3_tts_amd import kernels

    q, codes, scales, meta = _batch(device, 310, [2000, 5], [30, 1], hq=4, hkv=2, d=128, ps=16)
    need = kernels.paged_attention_int8_workspace_bytes(31, 2, 4, 2, 128)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=device)  # NaN partials, if one were read unwritten
    _check(q, codes, scales, meta, workspace=ws)
    with pytest.raises(ValueError):
        kernels.paged_attention_int8(q, codes, scales, meta, workspace=ws[:-1])
    with pytest.raises(TypeError):
        kernels.paged_attention_int8_workspace_bytes(31, 2, 34, 2, 128)


def test_rows_that_share_pages(nq, device):
    q, codes, scales, meta = _batch(device, 320, [64, 64, 50], None, hq=4, hkv=2, d=64, ps=16)
    meta.paged_kv_indices[4:8] = meta.paged_kv_indices[:4]
    _check(q, codes, scales, meta)


def test_blocks_that_were_never_written(nq, device):
    """A pool of zeros, scales too: every value is zero, and so is every output, masked keys or not."""

    for queries in (None, [5, 70, 2], [1, 33, 2]):
        q, codes, scales, meta = _batch(device, 330, [20, 70, 2], queries, hq=4, hkv=2, d=64, ps=64)
        codes.zero_()
        scales.zero_()
        assert not _check(q, codes, scales, meta).any()


@pytest.mark.parametrize("sm_scale", [0.0, 1e-38, -1e-30])
def test_scores_that_vanish(nq, device, sm_scale):
    """Factors of the scores down to zero, with blocks of zeros (scale 2^-126) among the keys: plain means."""

    for queries in (None, [40, 9]):
        q, codes, scales, meta = _batch(device, 331, [90, 40], queries, hq=4, hkv=2, d=128, ps=16)
        codes[meta.paged_kv_indices[1], 0] = 0
        scales[meta.paged_kv_indices[1], 0] = 2.0**-126
        _check(q, codes, scales, meta, sm_scale=sm_scale)


def test_page_outside_the_pool_beside_odd_scales(nq, device):
    """A skipped page takes nothing from the pool, whatever its first page holds."""

    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    for queries in (None, [30, 1]):
        q, codes, scales, meta = _batch(device, 332, [100, 40], queries, hq=4, hkv=2, d=64, ps=16)
        ids = meta.paged_kv_indices.cpu().numpy()
        ids = np.where(ids == 0, next(p for p in range(codes.shape[0]) if p not in ids), ids)
        ids[2] = codes.shape[0]
        meta.paged_kv_indices.copy_(torch.tensor(ids, dtype=torch.int32))
        outs = []
        for value in (1.0, -1.0, 0.0, float("nan"), float("-inf")):
            scales[0] = value
            status = torch.zeros(1, dtype=torch.int32, device=device)
            outs.append(paged_attention_int8(q, codes, scales, meta, status=status))
            assert int(status) == -1
        assert outs[0].isfinite().all()
        for out in outs[1:]:
            assert torch.equal(out.view(torch.int16), outs[0].view(torch.int16))


def test_many_rows(nq, device):
    """More rows than the kernels copy to LDS."""

    rng = np.random.default_rng(333)
    lens = rng.integers(0, 60, 700).tolist()
    _check(*_batch(device, 333, lens, None, hq=2, hkv=1, d=64, ps=16))
    queries = rng.integers(0, 4, 700).tolist()
    _check(*_batch(device, 334, lens, queries, hq=2, hkv=1, d=64, ps=16))


# -- scales that no value has ---------------------------------------------------------------------------


def _check_poisoned(device, queries, kind, value):
    """A visible block of vanishing probability whose scale of one kind and kv head is ``value``: the query heads of that kv
    head answer NaN, the others as before.  Row 0 (32 keys) lies in one decode span, row 1 (500) crosses several."""

    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    q, codes, scales, meta = _batch(device, 340, [32, 500], queries, hq=4, hkv=2, d=64, ps=16)
    q.fill_(1.0)
    first = [meta.paged_kv_indices[0], meta.paged_kv_indices[2]]  # the rows' first blocks: scores of -508
    for page in first:
        codes[page, 0], scales[page, 0] = -127, 2.0**-4
    want, bound = _want(q, codes, scales, meta, 1.0)
    for page in first:
        scales[page, kind, :, 0] = value
    out = paged_attention_int8(q, codes, scales, meta, sm_scale=1.0)
    assert out[:, :2].isnan().all()
    _compare(out[:, 2:], want[:, 2:], bound[:, 2:])


@pytest.mark.parametrize("queries", [None, [1, 1], [3, 40], [1, 40]])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_visible_scales_that_are_not_finite_answer_nan(nq, device, queries, kind, value):
    _check_poisoned(device, queries, kind, value)


@pytest.mark.parametrize("queries", [None, [3, 40]])
@pytest.mark.parametrize("kind", [0, 1])
def test_visible_negative_scales_answer_nan(nq, device, queries, kind):
    """No write leaves one: it is held to be as little a scale as infinity, in decode as in prefill."""

    _check_poisoned(device, queries, kind, -(2.0**-5))


def test_scales_that_are_no_powers_of_two(nq, device):
    """Any finite scale of at least zero is taken.  Prefill rounds V's code * scale to bf16, as the read back does: 2^-8 of
    sum P |v| more than the oracle's bound allows."""

    for queries in (None, [20, 70]):
        q, codes, scales, meta = _batch(device, 341, [90, 400], queries, hq=4, hkv=2, d=128, ps=16)
        scales.mul_(torch.rand(scales.shape, device=device) + 0.5)
        scales[meta.paged_kv_indices[1]] = 0.0
        want, bound = _want(q, codes, scales, meta)
        sizes, _ = _want(q, torch.stack((codes[:, 0], codes[:, 1].abs()), 1), scales, meta)
        from nari_qwen3_tts_amd.kernels import paged_attention_int8

        _compare(paged_attention_int8(q, codes, scales, meta), want, bound + (1 + 2.0**-6) * 2.0**-8 * sizes)


@pytest.mark.parametrize("keys,queries", [([60], None), ([600], None), ([60], [4]), ([600], [4]), ([600, 9], [4, 1])])
def test_scores_of_minus_infinity_answer_nan(nq, device, keys, queries):
    """A query whose every score is minus infinity has seen keys: NaN, as the softmax of the definition, whether its keys
    are read in one piece or in several; not the zeros of a query without keys."""

    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    q, codes, scales, meta = _batch(device, 342, keys, queries, hq=4, hkv=2, d=128, ps=16)
    codes[:, 0] = codes[:, 0].abs().clamp(1)
    want, bound = _want(q, codes, scales, meta)
    q[0, 1, 5] = float("-inf")
    out = paged_attention_int8(q, codes, scales, meta)
    assert out[0, 1].isnan().all()
    _compare(out[0, [0, 2, 3]], want[0, [0, 2, 3]], bound[0, [0, 2, 3]])
    _compare(out[1:], want[1:], bound[1:])


@pytest.mark.parametrize("old", [float("-inf"), float("inf"), float("nan"), -0.25])
def test_write_beside_a_scale_that_is_none(nq, device, old):
    """A block whose scale is not finite, or negative, stays unusable until a write at its first slot."""

    rng = np.random.default_rng(17)
    codes, scales = _pool(device, rng, 2, 16, 2, 64)
    scales[1, :, 0, 1] = old
    x = _bf16(rng, device, 2, 3, 2, 64)
    _check_write(codes, scales, x[0, :1], x[1, :1], *_slots(device, [1], [4]))
    assert scales[1, :, 0, 1].isnan().all() and scales[1, :, 0, 0].isfinite().all()
    _check_write(codes, scales, x[0], x[1], *_slots(device, [1, 1, 1], [0, 1, 2]))
    assert scales[1].isfinite().all()


@pytest.mark.parametrize("queries", [None, [3, 1, 20]])
@pytest.mark.parametrize("indptr", [[0, 3, 6, 9], [0, 4, 3, 6], [0, 6, 2, 2], [0, 6, 3, 1], [0, -5, 2, 6], [0, 6, 6, 0],
                                    [2, 1 << 30, 6, 6]])
def test_page_ranges_outside_the_list(nq, device, queries, indptr):
    """Ranges that decrease or pass the list's six pages set status; reads and writes stay inside the arguments (the workspace's
    partials included), and a call behind it is right."""

    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    q, codes, scales, meta = _batch(device, 350, [30, 40, 20], queries, hq=4, hkv=2, d=64, ps=16, spare=2)
    meta.paged_kv_indices = meta.paged_kv_indices[:6].clone()
    good = meta.paged_kv_indptr.clone()
    meta.paged_kv_indptr.copy_(torch.tensor(indptr, dtype=torch.int32))
    status = torch.zeros(1, dtype=torch.int32, device=device)
    paged_attention_int8(q, codes, scales, meta, status=status)
    assert int(status) == -1
    meta.paged_kv_indptr.copy_(good.clamp(max=6))
    _check(q, codes, scales, meta)


# -- one long prompt: tiles of 256 columns, eight waves ---------------------------------------------------


def _tile_columns(tokens, rows, hq, hkv, d):
    """Columns of a prefill tile, from the workspace: (tokens // (columns // group) + rows) tiles of each kv head, in 2 to 8
    pieces of a maximum, a sum and d values a column, or none where the pieces are one."""

    from nari_qwen3_tts_amd import _lib, kernels

    size = kernels.paged_attention_int8_workspace_bytes(tokens, rows, hq, hkv, d, _lib.NQ_ATTN_PREFILL)
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    found = {columns for columns in (128, 256) for pieces in range(2, 9)
             for n in [(tokens // (columns * hkv // hq) + rows) * hkv * pieces * columns]
             if up(8 * n) + up(4 * n * d) == size}
    assert len(found) == 1, "sizes whose workspace tells the tiles apart"
    return found.pop()


def _want_rows(q, codes, scales, meta):
    return o_kv.attention_rows(to_np(q), codes.cpu().numpy(), scales.cpu().numpy(), *(t.cpu().numpy() for t in (
        meta.paged_kv_indptr, meta.paged_kv_indices, meta.paged_kv_last_page_len, meta.qo_indptr)))


WIDE = [  # keys, queries, query heads, kv heads, page size
    ([1500], [1040], 16, 8, 16), ([1040], [1040], 16, 8, 64), ([2900], [1037], 16, 8, 16),
    ([900], [160], 16, 1, 16), ([100], [160], 16, 1, 64),  # the first 60 queries see no key
    ([800], [700], 6, 2, 16), ([730], [700], 6, 2, 64),  # a group that does not divide the columns
    ([700, 650], [700, 650], 16, 4, 128), ([500, 0, 300], [350, 1, 49], 16, 1, 16), ([2100], [2060], 4, 4, 32),
]


@pytest.mark.parametrize("case", range(len(WIDE)))
def test_prefill_of_a_long_prompt(nq, device, case):
    """Tiles of one piece, of two and of several; last tiles that are not full; empty rows and rows of one query beside."""

    from nari_qwen3_tts_amd import _lib
    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    keys, queries, hq, hkv, ps = WIDE[case]
    q, codes, scales, meta = _batch(device, 360 + case, keys, queries, hq=hq, hkv=hkv, d=128, ps=ps, tail=2)
    assert _tile_columns(q.shape[0], len(keys), hq, hkv, 128) == 256
    want, bound = _want_rows(q, codes, scales, meta)
    for parts in (_lib.NQ_ATTN_PREFILL, None):
        outs = []
        for _ in range(2):
            outs.append(torch.full_like(q, 7.0))
            paged_attention_int8(q, codes, scales, meta, parts=parts, out=outs[-1])
        _compare(outs[0], want, bound, f"{WIDE[case]}")
        assert (outs[0][sum(queries):] == 7.0).all()
        assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))


@pytest.mark.parametrize("hq,hkv,ps,keys,queries", [(16, 8, 16, 1500, 1040), (16, 1, 64, 900, 160), (6, 2, 16, 800, 700)])
def test_prefill_of_a_long_prompt_with_odd_blocks(nq, device, hq, hkv, ps, keys, queries):
    """A page outside the pool among the keys, blocks of NaN and infinite scales that the last queries alone see, codes and
    scales in other orders, queries and outputs as slices."""

    from nari_qwen3_tts_amd import _lib
    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    q, codes, scales, meta = _batch(device, 380 + hq, [keys], [queries], hq=hq, hkv=hkv, d=128, ps=ps)
    assert _tile_columns(queries, 1, hq, hkv, 128) == 256
    meta.paged_kv_indices[3] = codes.shape[0] + 7
    want, bound = _want_rows(q, codes, scales, meta)
    late = keys - 37  # a block that the last 37 queries see, a whole tile and a part of one behind
    page, block = int(meta.paged_kv_indices[late // ps]), late % ps // 16
    first = late // 16 * 16 - (keys - queries)  # the first query that sees it
    scales[page, 0, block], scales[page, 1, block] = float("nan"), 2.0**-5
    other = late + 16
    page, block = int(meta.paged_kv_indices[other // ps]), other % ps // 16
    scales[page, 1, block] = float("inf")
    packed = torch.zeros(queries, hq + 3, 128, dtype=torch.bfloat16, device=device)
    packed[:, 1:hq + 1] = q
    out = torch.full((queries, 2, hq, 128), 7.0, dtype=torch.bfloat16, device=device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    heads_first = codes.transpose(2, 3).contiguous().transpose(2, 3)
    blocks_last = scales.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0)
    paged_attention_int8(packed[:, 1:hq + 1], heads_first, blocks_last, meta, parts=_lib.NQ_ATTN_PREFILL, status=status,
                         out=out[:, 1])
    assert int(status) == -1 and (out[:, 0] == 7.0).all()
    assert out[first:, 1].isnan().all()
    _compare(out[:first, 1], want[:first], bound[:first])


def test_prefill_of_a_long_prompt_in_a_graph(nq, device):
    """Captured, replayed with other queries, keys and lengths, eager work between."""

    from nari_qwen3_tts_amd.kernels import paged_attention_int8

    q, codes, scales, meta = _batch(device, 390, [1300], [1040], hq=16, hkv=8, d=128, ps=16)
    assert _tile_columns(1040, 1, 16, 8, 128) == 256
    out = torch.zeros_like(q)
    paged_attention_int8(q, codes, scales, meta, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_attention_int8(q, codes, scales, meta, out=out)
    for last in (4, 1, 16, 9):
        q.normal_()
        codes.random_(-127, 128)
        meta.paged_kv_last_page_len.fill_(last)
        meta.qo_indptr[1] = 1000 + last
        want = paged_attention_int8(q, codes, scales, meta, out=torch.full_like(q, 7.0))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)) and want[:1000 + last].isfinite().all()

"""The 8-bit operators as a decoder layer's attention block uses them: row quantisation, int8 qkv projection, QK norm
and rotation, cache write, attention, row quantisation, int8 output projection; a prompt, then captured single-token
steps with a padding row.  Each stage is checked against its float64 oracle on the stage's own inputs."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from helpers import DecodeKey, PrefillKey, adopt_random, make_kv, to_np
from oracle import int8 as o_int8
from oracle import kv_int8 as o_kv

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, D, PS = 256, 4, 2, 64, 32
WIDTH = (HQ + 2 * HKV) * D


class Layer:
    def __init__(self, nq, device, rng):
        from nari_qwen3_tts_amd import layers

        def bf16(*shape, size=1.0, mean=0.0):
            return torch.tensor(mean + size * rng.standard_normal(shape), dtype=torch.bfloat16, device=device)

        self.w_qkv, self.s_qkv = layers.quantize_int8_rows(bf16(WIDTH, HIDDEN, size=0.06))
        self.w_o, self.s_o = layers.quantize_int8_rows(bf16(HIDDEN, HQ * D, size=0.06))
        self.q_norm, self.k_norm = bf16(D, size=0.2, mean=1.0), bf16(D, size=0.2, mean=1.0)

    def __call__(self, x, pool, slots, meta, positions, stages=None):
        from nari_qwen3_tts_amd import kernels, layers

        codes, scales = layers.quantize_int8_rows(x)
        qkv = layers.linear_int8(codes, scales, self.w_qkv, self.s_qkv)
        if stages is not None:
            stages.update(codes=codes, scales=scales, qkv=qkv.clone(), before=[t.clone() for t in pool])
        heads = qkv.view(-1, HQ + 2 * HKV, D)
        q, k, v = heads[:, :HQ], heads[:, HQ:HQ + HKV], heads[:, HQ + HKV:]
        kernels.paired_qk_norm_rope_(q, k, self.q_norm, self.k_norm, positions, 1e-6, 1e4)
        kernels.paged_cache_write_int8_(k, v, *pool, *slots)
        mixed = kernels.paged_attention_int8(q, *pool, meta)
        codes, scales = layers.quantize_int8_rows(mixed.view(-1, HQ * D))
        out = layers.linear_int8(codes, scales, self.w_o, self.s_o)
        if stages is not None:
            stages.update(q=q, k=k, v=v, mixed=mixed, codes_o=codes, scales_o=scales)
        return out


def _check_rows(x, codes, scales):
    want, want_s = o_int8.quantize_rows(to_np(x))
    assert np.array_equal(codes.cpu().numpy(), want)
    # one fp32 division
    assert np.all(np.abs(scales.cpu().numpy().astype(np.float64) - want_s) <= 2.0**-24 * want_s)


def _check_product(out, codes, scales, w, sw):
    want = o_int8.linear(*(t.cpu().numpy() for t in (codes, scales, w, sw)))
    # the sum to fp32 and two products (2^-24 each), the result to bf16 (2^-8)
    assert np.all(np.abs(to_np(out) - want) <= np.abs(want) * (2.0**-8 + 4 * 2.0**-24))


def _check_stages(layer, x, pool, slots, meta, out, s):
    _check_rows(x, s["codes"], s["scales"])
    _check_product(s["qkv"], s["codes"], s["scales"], layer.w_qkv, layer.s_qkv)
    codes, scales = (t.cpu().numpy() for t in s["before"])
    o_kv.write(codes, scales, to_np(s["k"]), to_np(s["v"]), *(t.cpu().numpy() for t in slots))
    assert np.array_equal(pool[0].cpu().numpy(), codes) and np.array_equal(pool[1].cpu().numpy(), scales)
    metadata = [None if t is None else t.cpu().numpy() for t in (
        meta.paged_kv_indptr, meta.paged_kv_indices, meta.paged_kv_last_page_len, meta.qo_indptr)]
    want, bound = o_kv.attention(to_np(s["q"]), codes, scales, *metadata)
    assert np.all(np.abs(to_np(s["mixed"]) - want) <= bound)
    _check_rows(s["mixed"].reshape(-1, HQ * D), s["codes_o"], s["scales_o"])
    _check_product(out, s["codes_o"], s["scales_o"], layer.w_o, layer.s_o)


def test_prompt_and_captured_steps(nq, device):
    rng = np.random.default_rng(400)
    layer = Layer(nq, device, rng)
    prompts, steps, rows = [40, 1, 17], 36, 4  # the last row is padding: one token in a page of its own
    pages = [-(-(n + steps) // PS) for n in prompts]
    order = rng.permutation(sum(pages) + 1)
    scratch, table, at = int(order[-1]), [], 0
    for n in pages:
        table.append(order[at:at + n])
        at += n
    pool = (torch.zeros(sum(pages) + 1, 2, PS, HKV, D, dtype=torch.int8, device=device),
            torch.zeros(sum(pages) + 1, 2, PS // 16, HKV, device=device))

    def int32(x):
        return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)

    def int64(x):
        return torch.tensor(np.asarray(x), dtype=torch.long, device=device)

    def tokens(n):
        return torch.tensor(rng.standard_normal((n, HIDDEN)), dtype=torch.bfloat16, device=device)

    # the prompt
    used = [-(-n // PS) for n in prompts]
    meta = SimpleNamespace(
        qo_indptr=int32(np.concatenate(([0], np.cumsum(prompts)))), paged_kv_indptr=int32(np.concatenate(([0], np.cumsum(used)))),
        paged_kv_indices=int32(np.concatenate([t[:u] for t, u in zip(table, used)])),
        paged_kv_last_page_len=int32([(n - 1) % PS + 1 for n in prompts]))
    where = np.concatenate([np.arange(n) for n in prompts])
    slots = (int64(np.concatenate([table[r][np.arange(n) // PS] for r, n in enumerate(prompts)])), int64(where % PS))
    x, stages = tokens(sum(prompts)), {}
    out = layer(x, pool, slots, meta, int64(where), stages)
    _check_stages(layer, x, pool, slots, meta, out, stages)

    # single-token steps: the buffers a captured step reads, filled in place
    x = tokens(rows)
    meta = SimpleNamespace(qo_indptr=None, paged_kv_indptr=int32(np.zeros(rows + 1)),
                           paged_kv_indices=int32(np.zeros(sum(pages) + 1)), paged_kv_last_page_len=int32(np.ones(rows)))
    slots, positions = (int64(np.zeros(rows)), int64(np.zeros(rows))), int64(np.zeros(rows))

    def plan(step):
        lens = [n + step + 1 for n in prompts]
        used = [-(-n // PS) for n in lens] + [1]
        ids = np.concatenate([t[:u] for t, u in zip(table, used)] + [[scratch]])
        meta.paged_kv_indices[:len(ids)].copy_(int32(ids))
        meta.paged_kv_indptr.copy_(int32(np.concatenate(([0], np.cumsum(used)))))
        meta.paged_kv_last_page_len.copy_(int32([(n - 1) % PS + 1 for n in lens] + [1]))
        last = np.array([n - 1 for n in lens] + [0])
        slots[0].copy_(int64([table[r][last[r] // PS] for r in range(3)] + [scratch]))
        slots[1].copy_(int64(last % PS))
        positions.copy_(int64(last))
        x.copy_(tokens(rows))

    plan(0)
    kept = [t.clone() for t in pool]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer(x, pool, slots, meta, positions)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = layer(x, pool, slots, meta, positions)
    for t, k in zip(pool, kept):
        t.copy_(k)
    for step in range(steps):
        plan(step)
        eager, stages = [t.clone() for t in pool], {}
        out = layer(x, eager, slots, meta, positions, stages)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(replayed.view(torch.int16), out.view(torch.int16))
        assert torch.equal(pool[0], eager[0]) and torch.equal(pool[1], eager[1])
        if step % 7 == 0:
            _check_stages(layer, x, pool, slots, meta, out, stages)


def test_side_stream_behind_its_inputs(nq, device):
    """Every launch goes to the current stream: work queued there before and after is ordered with it."""

    from nari_qwen3_tts_amd import kernels, layers

    rng = np.random.default_rng(401)
    layer = Layer(nq, device, rng)
    source = torch.tensor(rng.standard_normal((5, HIDDEN)), dtype=torch.bfloat16, device=device)
    meta = SimpleNamespace(
        qo_indptr=None, paged_kv_indptr=torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32, device=device),
        paged_kv_indices=torch.arange(5, dtype=torch.int32, device=device),
        paged_kv_last_page_len=torch.ones(5, dtype=torch.int32, device=device))
    slots = torch.arange(5, device=device), torch.zeros(5, dtype=torch.long, device=device)
    pools = [(torch.zeros(5, 2, PS, HKV, D, dtype=torch.int8, device=device),
              torch.zeros(5, 2, PS // 16, HKV, device=device)) for _ in range(2)]
    want = layer(source, pools[0], slots, meta, slots[1])
    keys, values = kernels.paged_cache_read_int8(*pools[0], *slots)
    torch.cuda.synchronize()
    stream, busy = torch.cuda.Stream(), torch.zeros(1 << 26, device=device)
    x = torch.full_like(source, float("nan"))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(20):
            busy.add_(1.0)
        x.copy_(source)
        out = layer(x, pools[1], slots, meta, slots[1])
        again = kernels.paged_cache_read_int8(*pools[1], *slots)
        result = [t.clone() for t in (out, *again)]
    stream.synchronize()
    for got, expected in zip(result, (want, keys, values)):
        assert torch.equal(got, expected)


def test_two_graphs_with_one_workspace(nq, device):
    """Two captured calls that share a workspace, replayed one behind the other in either order."""

    from nari_qwen3_tts_amd import kernels

    rng = np.random.default_rng(402)
    pool = (torch.tensor(rng.integers(-127, 128, (70, 2, 16, HKV, D)), dtype=torch.int8, device=device),
            torch.full((70, 2, 1, HKV), 2.0**-6, device=device))
    metas = [SimpleNamespace(
        qo_indptr=qo, paged_kv_indptr=torch.tensor(indptr, dtype=torch.int32, device=device),
        paged_kv_indices=torch.tensor(rng.permutation(70), dtype=torch.int32, device=device),
        paged_kv_last_page_len=torch.tensor([7, 16], dtype=torch.int32, device=device))
        for qo, indptr in ((None, [0, 40, 65]), (torch.tensor([0, 50, 51], dtype=torch.int32, device=device), [0, 60, 70]))]
    queries = [torch.tensor(rng.standard_normal((n, HQ, D)), dtype=torch.bfloat16, device=device) for n in (2, 51)]
    need = max(kernels.paged_attention_int8_workspace_bytes(q.shape[0], 2, HQ, HKV, D) for q in queries)
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    outs, graphs = [torch.empty_like(q) for q in queries], []

    def call(i, out):
        return kernels.paged_attention_int8(queries[i], *pool, metas[i], workspace=workspace, out=out)

    for i in range(2):
        call(i, outs[i])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            call(i, outs[i])
    for turn in ((0, 1), (1, 0), (0, 1, 0), (1, 1, 0)):
        for q in queries:
            q.copy_(torch.tensor(rng.standard_normal(q.shape), dtype=torch.bfloat16, device=device))
        want = [kernels.paged_attention_int8(queries[i], *pool, metas[i]) for i in range(2)]
        workspace.fill_(255)  # NaN partials, if one were read unwritten
        for i in turn:
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in set(turn):
            assert torch.equal(outs[i].view(torch.int16), want[i].view(torch.int16))


@pytest.mark.parametrize("prefill", [False, True])
def test_captured_steps_with_the_planner(nq, device, prefill):
    """Write and attention on the metadata of the framework's own planner, captured with requests of one token (as a capture
    slot is warmed) and replayed with others: longer histories, more pages, padding rows and padding tokens."""

    from nari_qwen3_tts_amd import _lib, kernels

    rng = np.random.default_rng(403 + prefill)
    kv = make_kv(nq, device, hq=HQ, hkv=HKV, d=D, pages=96, ps=PS, scratch=5)
    key = PrefillKey(5, 60) if prefill else DecodeKey(5)
    ctx = kv.create_prefill(key, slot=0) if prefill else kv.create_decode(key, slot=0)
    pubs = kv.prepare_capture(ctx, key)
    meta, tokens = ctx.metadata, ctx.token_capacity
    parts = _lib.NQ_ATTN_PREFILL if prefill else _lib.NQ_ATTN_DECODE
    codes = torch.tensor(rng.integers(-127, 128, (96, 2, PS, HKV, D)), dtype=torch.int8, device=device)
    scales = torch.tensor(2.0 ** rng.integers(-9, -4, (96, 2, PS // 16, HKV)), dtype=torch.float32, device=device)
    x = torch.zeros(tokens, HQ + 2 * HKV, D, dtype=torch.bfloat16, device=device)
    out = torch.zeros(tokens, HQ, D, dtype=torch.bfloat16, device=device)
    status = torch.zeros(1, dtype=torch.int32, device=device)

    def step():
        kernels.paged_cache_write_int8_(x[:, HQ:HQ + HKV], x[:, HQ + HKV:], codes, scales, meta.write_pages,
                                        meta.write_offsets, status)
        kernels.paged_attention_int8(x[:, :HQ], codes, scales, meta, parts=parts, status=status, out=out)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    kv.finish_capture(ctx, pubs)

    rids = tuple(adopt_random(kv, rng, [300, 3, 120]))
    for turn in range(4):
        news = [int(n) for n in rng.integers(1, 20, 3)]
        pubs = kv.prepare_prefill(ctx, key, rids, news) if prefill else kv.prepare_decode(ctx, key, rids)
        x.copy_(torch.tensor(rng.standard_normal(x.shape), dtype=torch.bfloat16, device=device))
        want_c, want_s = codes.cpu().numpy(), scales.cpu().numpy()
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert int(status) == 0
        now = ctx.metadata
        live = sum(news) if prefill else 3
        pages, offsets = now.write_pages.cpu().numpy(), now.write_offsets.cpu().numpy()
        heads = to_np(x)
        o_kv.write(want_c, want_s, heads[:, HQ:HQ + HKV], heads[:, HQ + HKV:], pages, offsets)
        got_c, got_s = codes.cpu().numpy(), scales.cpu().numpy()
        held = [p for p in range(96) if p not in kv._scratch_pages]
        assert np.array_equal(got_c[held], want_c[held]) and np.array_equal(got_s[held], want_s[held])
        want, bound = o_kv.attention(heads[:, :HQ], got_c, got_s, *(
            None if t is None else t.cpu().numpy() for t in (
                now.paged_kv_indptr, now.paged_kv_indices, now.paged_kv_last_page_len, now.qo_indptr)))
        assert np.all(np.abs(to_np(out)[:live] - want[:live]) <= bound[:live]), turn
        if prefill:
            assert (out[live:] == 7.0).all()
        for p in pubs:
            p.publish()

"""The 4-bit cache behind the executor: a serving run (packed prefill, prefix hit with a chunk, decode
steps, the fused prologue, drafted tokens) and a captured decode step, against the 64-bit statement on the
bytes that the pool holds."""

import math

import pytest
import torch

from llama_lite_npu_b200 import kernels, workloads as W
from llama_lite_npu_b200.cuda_graph import CudaGraphRunner
from llama_lite_npu_b200.executor import PagedKVExecutor
from llama_lite_npu_b200.paged_attention import PagedKVCacheManager
from oracle import kv4_oracle as K4

SCALE = 1.0 / math.sqrt(128)
LOG2E = 1.4426950408889634
U = 2.0 ** -11
DEV = "cuda:0"


def test_manager_and_executor_formats_on_the_host():
    mgr = PagedKVCacheManager(2, 3, 128, 5, 16, torch.float16, "cpu", kv_format="kv4")
    assert [tuple(b.shape) for b in mgr.gpu_kv_buffer] == [(5, 6, 1152)] * 2 and mgr.max_tokens == 80
    assert mgr.gpu_kv_buffer[0].dtype == torch.uint8 and mgr.alloc(20).tolist() == [0, 1]
    assert PagedKVCacheManager(1, 1, 128, 2, 16, torch.float16, "cpu").kv_format == "fp16"
    for bad in (dict(kv_format="int4"), dict(kv_format="kv4", head_dim=64), dict(kv_format="kv4", page_size=32)):
        args = dict(num_layers=1, num_kv_heads=1, head_dim=128, num_pages=2, page_size=16, device="cpu")
        args.update(bad)
        with pytest.raises(ValueError):
            PagedKVCacheManager(**args)
    ex = PagedKVExecutor(1, 1, 128, 8, 4, 64, device="cpu", kv_format="kv4")
    ids = ex.reserve_paged_requests([20, 3])
    ex.activate_paged_packed_prefill_batch(ids, [20, 3])
    assert ex.atten_info.kv_buffer[0].shape == (8, 2, 1152)


def _attend(ex, xq, layer, req_ids, starts, ctx, qlen):
    """Oracle outputs and error bounds (counted as in test_gpu_kv4.py) for the rows of a batch."""
    pool = ex.kv_mem_manager.gpu_kv_buffer[layer].cpu()
    table = ex.req_tokens_manager.b_req_tokens_table.cpu()
    kvh = pool.shape[1] // 2
    out = torch.zeros(xq.shape, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for r, s, c, n in zip(req_ids, starts, ctx, qlen):
        x = K4.rows_of(pool, table[r, : c + n])
        o, mag, dot = K4.attention(xq[s: s + n].cpu(), x[:, :kvh], x[:, kvh:], c, SCALE)
        out[s: s + n] = o
        tol[s: s + n] = (U * o.abs() + 2.0 ** -25 + (2 * U + 2.0 ** -18 + 2.0 ** -19 * dot + 2 * U * dot) * mag
                         + (c + n) * 2.0 ** -24 * x[:, kvh:].abs().max())
    return out, tol


def _check(got, want):
    out, tol = want
    assert float(((got.cpu().double() - out).abs() - tol).max()) <= 0


@pytest.mark.gpu
def test_serving_scenario_on_a_4_bit_cache(built_lib):
    kvh, heads, layers = 2, 8, 2
    ex = PagedKVExecutor(layers, kvh, 128, 256, 8, 512, page_size=16, device=DEV, kv_format="kv4")
    for buf in ex.kv_mem_manager.gpu_kv_buffer:
        buf.fill_(0xFF)                                          # unwritten slots read as NaN
    rand = lambda n, h, stream: W.hash_normal_fp16(99, (n, h, 128), stream).to(DEV)  # noqa: E731
    prompts = [list(range(1000, 1000 + n)) for n in (70, 33, 150)]
    ids = ex.reserve_paged_requests([len(p) for p in prompts])
    ex.activate_paged_packed_prefill_batch(ids, [len(p) for p in prompts])
    for layer in range(layers):
        xq, xk, xv = rand(253, heads, 10 + layer), rand(253, kvh, 20 + layer), rand(253, kvh, 30 + layer)
        got = ex.context_forward(xq, xk, xv, layer, SCALE * LOG2E)
        _check(got, _attend(ex, xq, layer, ids, [0, 70, 103], [0, 0, 0], [70, 33, 150]))
    ex.store_paged_request_prefix(prompts[2], ids[2], first_token_id=5)
    ex.release_paged_request_ids((ids[1],))
    shared = ex.req_tokens_manager.request_pages(ids[2])[:9]
    before = ex.kv_mem_manager.gpu_kv_buffer[0][list(shared)].clone()

    # a prefix hit: 144 tokens of history, a chunk of 40, through the fused prologue
    rid, matched, _ = ex.share_paged_prefix_from_cache(prompts[2][:144] + list(range(5000, 5040)))
    assert matched == 144
    ex.activate_paged_chunk_prefill_batch((rid,), [144], [40])
    w = (1 + 0.1 * W.hash_normal_fp16(98, (128,), 1).float()).half().to(DEV)
    ang = W.hash_normal_fp16(98, (40, 64), 2).float()
    cos, sin = (torch.cat((f(ang), f(ang)), 1).half().to(DEV) for f in (torch.cos, torch.sin))
    for layer in range(layers):
        xq, xkv = rand(40, heads, 40 + layer), rand(40, 2 * kvh, 50 + layer).flatten(1)
        q_want = K4.norm_rope(xq.cpu(), w.cpu(), 1e-6, cos.cpu(), sin.cpu())
        got = ex.fused_context_forward(xq, xkv, w, w, 1e-6, cos, sin, layer, SCALE * LOG2E)
        assert float((xq.cpu().float() - q_want.float()).abs().max()) <= 2e-2     # rotated in place
        _check(got, _attend(ex, xq, layer, [rid], [0], [144], [40]))
    assert torch.equal(ex.kv_mem_manager.gpu_kv_buffer[0][list(shared)], before)   # shared pages untouched

    batch = (ids[2], ids[0], rid)
    for step in range(3):
        ex.extend_paged_requests_on_device(batch)
        lens = [ex.req_tokens_manager.req_token_count[r] for r in batch]
        for layer in range(layers):
            xq = rand(3, heads, 70 + step)
            if step < 2:
                got = ex.token_forward(xq, rand(3, kvh, 80 + step), rand(3, kvh, 90 + step), layer, SCALE)
            else:
                got = ex.fused_token_forward(xq, rand(3, 2 * kvh, 95).flatten(1), w, w, 1e-6, cos[:3], sin[:3], layer, SCALE)
            _check(got, _attend(ex, xq, layer, batch, [0, 1, 2], [n - 1 for n in lens], [1, 1, 1]))

    # five drafted tokens per request verified in one pass
    ctx = [ex.req_tokens_manager.req_token_count[r] for r in batch]
    ex.activate_paged_chunk_prefill_batch(batch, ctx, [5, 5, 5])
    for layer in range(layers):
        xq = rand(15, heads, 110 + layer)
        got = ex.context_forward(xq, rand(15, kvh, 120), rand(15, kvh, 130), layer, SCALE * LOG2E)
        _check(got, _attend(ex, xq, layer, batch, [0, 5, 10], ctx, [5, 5, 5]))
    ex.release_paged_request_ids(batch)
    kernels.check_status(0)


@pytest.mark.gpu
@pytest.mark.parametrize("extend", ["extend_paged_requests", "stage_paged_decode_step"])
def test_4_bit_decode_step_replays_in_a_graph(extend, built_lib):
    """The captured step (advance, quantising append and decode of two layers) equals an eager twin: the pools
    byte for byte, the outputs within the length bucket's different cut."""
    kvh, heads, layers = 2, 16, 2
    ex, ref = (PagedKVExecutor(layers, kvh, 128, 512, 8, 1024, page_size=16, device=DEV, kv_format="kv4") for _ in range(2))
    for e in (ex, ref):
        for li, buf in enumerate(e.kv_mem_manager.gpu_kv_buffer):
            slots = torch.arange(512 * 16, dtype=torch.int32, device=DEV)
            kernels.update_kv_buffer_kv4(W.hash_normal_fp16(5 + li, (512 * 16, 2 * kvh, 128), 1).to(DEV), slots, buf)
    ids = ex.reserve_paged_requests([37, 100, 64, 5])
    assert ref.reserve_paged_requests([37, 100, 64, 5]) == ids

    def model_on(executor):
        class Model:
            def forward(self, input_ids, position_ids, info):
                saved, executor.atten_info = executor.atten_info, info
                try:
                    x = xq
                    for layer in range(layers):
                        x = executor.token_forward(x, xk, xv, layer, SCALE)
                    return x
                finally:
                    executor.atten_info = saved
        return Model()

    runner, eager = CudaGraphRunner(model_on(ex), "harness"), model_on(ref)
    xq = torch.empty(4, heads, 128, dtype=torch.float16, device=DEV)
    xk, xv = torch.empty(4, kvh, 128, dtype=torch.float16, device=DEV), torch.empty(4, kvh, 128, dtype=torch.float16, device=DEV)
    inp = torch.zeros(4, 1, dtype=torch.long, device=DEV)
    for step in range(18):
        getattr(ex, extend)(ids)
        ref.extend_paged_requests(ids)
        for i, t in enumerate((xq, xk, xv)):
            t.copy_(W.hash_normal_fp16(50 + step, tuple(t.shape), i))
        want = eager.forward(inp, inp, ref.atten_info).clone()
        got = runner(inp, inp, ex.atten_info)
        torch.cuda.synchronize()
        assert float((got.float() - want.float()).abs().max()) <= 2e-3, step
        assert torch.equal(ex.atten_info.b_seq_len.cpu(), ref.atten_info.b_seq_len.cpu())
    for a, b in zip(ex.kv_mem_manager.gpu_kv_buffer, ref.kv_mem_manager.gpu_kv_buffer):
        assert torch.equal(a, b)
    assert (runner.replay_count, runner.fallback_count) == (18, 0)
    kernels.check_status(0)


@pytest.mark.gpu
def test_4_bit_decode_step_never_synchronises_with_the_host(built_lib):
    ex = PagedKVExecutor(1, 2, 128, 128, 8, 512, page_size=16, device=DEV, kv_format="kv4")
    ids = ex.reserve_paged_requests([30, 47, 5])
    ex.extend_paged_requests(ids)
    xq = torch.zeros(3, 8, 128, dtype=torch.float16, device=DEV)
    xk = torch.zeros(3, 2, 128, dtype=torch.float16, device=DEV)
    xkv = torch.zeros(3, 512, dtype=torch.float16, device=DEV)
    w, cos = torch.ones(128, dtype=torch.float16, device=DEV), torch.ones(3, 128, dtype=torch.float16, device=DEV)
    ex.token_forward(xq, xk, xk, 0, SCALE)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(20):
            ex.extend_paged_requests_on_device(ids)
            ex.token_forward(xq, xk, xk, 0, SCALE)
            ex.fused_token_forward(xq, xkv, w, w, 1e-6, cos, cos, 0, SCALE)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    torch.cuda.synchronize()
    kernels.check_status(0)

"""The 4-bit paged cache on the GPU, at the calls that the documentation allows and that are easy to get wrong: large
pools, wide tables, garbage in places never written, side streams and branches of one capture, a first call
inside a capture, many requests, the same slot twice, lengths that change under a captured graph.

Errors are counted as in test_gpu_kv4.py; where two calls do the same arithmetic they are held to equal bits."""

import gc
import math
import os
import subprocess
import sys

import pytest
import torch

from llama_lite_npu_b200 import _lib, kernels
from oracle import kv4_oracle as K4
from test_gpu_kv4 import DEV, LOG2E, SCALE, Case, _randn, _slots, _within

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module", autouse=True)
def _lib_loaded(built_lib):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    yield
    kernels.check_status(0)


# The largest and smallest scales and every kind of special fp16 number, both signs.
GARBAGE = torch.tensor([0x7BFF, -0x8000 + 0x7BFF, 0x7C00, -0x8000 + 0x7C00, 0x7E01, -0x8000 + 0x7E01, 1, -0x8000],
                       dtype=torch.int32).to(torch.int16)


@pytest.mark.parametrize("lens, q_lens, qh, kvh", [([1, 130, 33], [1, 130, 5], 4, 2), ([150, 7], [7, 3], 8, 1),
                                                   ([263], [260], 2, 1), ([97, 45], [1, 1], 16, 2)])
@pytest.mark.parametrize("kind", range(8))
def test_places_never_written_may_hold_anything(lens, q_lens, qh, kvh, kind):
    c = Case(sum(lens) + kind, lens, qh, kvh, q_lens)
    clean = c.prefill().clone()
    want, tol_d, tol_p = c.want()
    fill = torch.full_like(c.pool, 0x0F if kind & 1 else 0xF0)
    fill.view(torch.int16)[..., 512:] = GARBAGE[kind]
    for i in range(len(lens)):
        _take(fill, c.pool, c.slots[i])
    got = c.prefill(pool=fill.to(DEV))
    assert torch.equal(got, clean)
    _within(got, want, tol_p)
    if max(q_lens) == 1:
        c.pool = fill
        _within(c.decode(), want, tol_d)


def _take(dst, src, slots):
    """The given slots' codes and scales of src into dst."""
    for s in slots.tolist():
        page, t = divmod(s, 16)
        dst[page][:, 64 * t: 64 * t + 64] = src[page][:, 64 * t: 64 * t + 64]
        dst[page][:, 1024 + 8 * t: 1032 + 8 * t] = src[page][:, 1024 + 8 * t: 1032 + 8 * t]


@pytest.mark.parametrize("n, kvh", [(2371, 8), (4742, 3)])
def test_long_appends_take_four_rows_per_warp(n, kvh):
    """Enough tokens for four rows per warp, a last quad of three tokens, and heads that do not divide by four."""
    x = _randn(n, (n, 2 * kvh, 128), 1)
    pages = (n + 15) // 16 + 2
    slots = _slots(n, n, pages * 16)
    slots[11] = -5
    want = torch.zeros(pages, 2 * kvh, K4.BLOCK, dtype=torch.uint8)
    K4.append(x, slots, want)
    pool = torch.zeros_like(want).to(DEV)
    kernels.update_kv_buffer_kv4(x.to(DEV), slots.to(DEV), pool)
    with pytest.raises(RuntimeError, match="slot_mapping"):
        kernels.check_status(0)
    assert torch.equal(pool.cpu(), want)
    slots[11] = slots[12]
    many = slots.repeat(3)                     # the same slots several times in one read-back
    back = kernels.gather_kv_buffer_kv4(pool, many.to(DEV))
    assert torch.equal(back.cpu(), K4.rows_of(want, slots).half().repeat(3, 1, 1))


@pytest.mark.parametrize("n, qh, kvh", [(1901, 10, 5), (477, 64, 8)])
def test_long_fused_appends_equal_short_ones(n, qh, kvh):
    """One launch over many tokens (four rows per warp) and launches over a few (one row) write the same bytes."""
    xq, xkv = _randn(n, (n, qh, 128), 1).to(DEV), _randn(n, (n, 2 * kvh * 128), 2).to(DEV)
    wq, wk = ((1 + 0.3 * _randn(n, (128,), s).float()).half().to(DEV) for s in (3, 4))
    ang = 3.0 * _randn(n, (n, 64), 5).float()
    cos, sin = ang.cos().half().to(DEV), ang.sin().half().to(DEV)
    pages = (n + 15) // 16 + 1
    slots = _slots(n, n, pages * 16).to(DEV)
    pools = [torch.zeros(pages, 2 * kvh, K4.BLOCK, dtype=torch.uint8, device=DEV) for _ in (0, 1)]
    outs = [torch.empty_like(xq) for _ in (0, 1)]
    kernels.fused_qk_norm_rope_append_kv4(xq, xkv, wq, wk, 1e-6, cos, sin, slots, pools[0], out=outs[0])
    for a in range(0, n, 37):
        z = slice(a, min(n, a + 37))
        kernels.fused_qk_norm_rope_append_kv4(xq[z], xkv[z], wq, wk, 1e-6, cos[z], sin[z], slots[z], pools[1], out=outs[1][z])
    assert torch.equal(pools[0], pools[1]) and torch.equal(outs[0], outs[1])
    kv = xkv.cpu().view(n, 2 * kvh, 128)
    c2, s2 = torch.cat((cos, cos), 1).cpu(), torch.cat((sin, sin), 1).cpu()
    rows = torch.cat((K4.norm_rope(kv[:, :kvh], wk.cpu(), 1e-6, c2, s2), kv[:, kvh:]), 1)
    want = torch.zeros(pages, 2 * kvh, K4.BLOCK, dtype=torch.uint8)
    K4.append(rows, slots.cpu(), want)
    # x * rrms is rounded to 32 bits before it is rounded to fp16: 2 half steps of 2^-24 against a spacing of ties of
    # 2^-11 move about 2^-11 of the elements of K by one step of fp16, which now and then moves a code by one or the
    # group's scale by one step (7 codes * 2^-10 of it).
    got, ref = K4.rows_of(pools[0].cpu(), slots.cpu()), K4.rows_of(want, slots.cpu())
    step = K4.quantise(rows)[1].double().repeat_interleave(32, -1)
    assert bool(((got - ref).abs() <= step * (1 + 2.0 ** -6)).all())
    assert torch.equal(got[:, kvh:], ref[:, kvh:])
    moved = ((got != ref).unflatten(-1, (4, 32)).any(-1)).double().mean()      # groups: 32 elements each
    assert float(moved) <= 32 * 2.0 ** -11


def test_same_slot_twice_with_identical_rows():
    x = _randn(3, (9, 4, 128))
    x[5], x[8] = x[2], x[2]
    slots = torch.tensor([0, 1, 30, 3, 4, 30, 6, 7, 30], dtype=torch.int32)
    want = torch.zeros(2, 4, K4.BLOCK, dtype=torch.uint8)
    K4.append(x, slots, want)
    for _ in range(20):
        pool = torch.zeros(2, 4, K4.BLOCK, dtype=torch.uint8, device=DEV)
        kernels.update_kv_buffer_kv4(x.to(DEV), slots.to(DEV), pool)
        assert torch.equal(pool.cpu(), want)


def test_offsets_past_32_bits():
    """The same sequences on the last pages of a pool of more than 2^32 bytes, whose page stride is odd in every
    sense the format allows, and in a small pool: equal bits from every operator."""
    kvh, qh, n_used = 4, 16, 40
    stride = 2 * kvh * K4.BLOCK + 48
    pages = (1 << 32) // stride + 3 * n_used
    base = torch.empty(pages * stride, dtype=torch.uint8, device=DEV)
    big = base.as_strided((pages, 2 * kvh, K4.BLOCK), (stride, K4.BLOCK, 1))
    small = torch.zeros(n_used, 2 * kvh, K4.BLOCK, dtype=torch.uint8, device=DEV)
    first = pages - n_used
    assert first * stride > 1 << 32
    big[first:] = 0
    lens = [300, 131, 17]
    n = sum(lens)
    xkv, xq = _randn(8, (n, 2 * kvh * 128), 1).to(DEV), _randn(8, (n, qh, 128), 2).to(DEV)
    ang = _randn(8, (n, 64), 3).float()
    cos, sin = ang.cos().half().to(DEV), ang.sin().half().to(DEV)
    block = torch.zeros(3, 20, dtype=torch.int32)
    at, slots = 0, []
    for i, m in enumerate(lens):
        np_ = (m + 15) // 16
        block[i, :np_] = torch.arange(at, at + np_)
        slots.append(torch.arange(at * 16, at * 16 + m))
        at += np_
    slots = torch.cat(slots).int().to(DEV)
    block = block.to(DEV)
    res = []
    for pool, off in ((small, 0), (big, first)):
        s = (slots.long() + off * 16).int()
        tbl = (block.long() + off).int()
        tok = (tbl.unsqueeze(-1) * 16 + torch.arange(16, device=DEV, dtype=torch.int32)).flatten(1).contiguous()
        kernels.update_kv_buffer_kv4(xkv.view(n, 2 * kvh, 128), s, pool)
        got = [kernels.gather_kv_buffer_kv4(pool, s)]
        out = torch.empty_like(xq)
        kernels.fused_qk_norm_rope_append_kv4(xq, xkv, None, None, 1e-6, cos, sin, s, pool, out=out)
        got += [out, kernels.gather_kv_buffer_kv4(pool, s)]
        ln = torch.tensor(lens, device=DEV)
        for kind, t in (("block", tbl), ("token", tok)):
            got.append(kernels.flash_decoding_kv4(xq[:3], pool, SCALE, t, ln, max(lens), table_kind=kind))
            for ql in ([3, 1, 2], [200, 131, 1]):
                qd = torch.tensor(ql, device=DEV)
                got.append(kernels.paged_chunk_flash_attention_kv4(
                    xq[: sum(ql)], pool, SCALE * LOG2E, t, torch.arange(3, dtype=torch.int32, device=DEV),
                    (qd.cumsum(0) - qd).int(), ln - qd, qd, max(ql), table_kind=kind))
        res.append(got)
    kernels.check_status(0)
    for a, b in zip(*res):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())
    assert torch.equal(big[first:].cpu(), small.cpu())


def test_wide_strided_tables_and_rows_behind_the_last_sequence():
    c = Case(17, [70, 33], 8, 2, [5, 3])
    wide = torch.full((c.block.shape[0], 2 * c.block.shape[1] + 5), -7, dtype=torch.int32)
    wide[:, : c.block.shape[1]] = c.block
    tbl = wide.to(DEV)[:, : c.block.shape[1]]
    want, _, tol = c.want()
    pad = torch.cat((c.q, torch.full((6, 8, 128), float("nan"), dtype=torch.float16))).to(DEV)
    ql = torch.tensor(c.q_lens)
    args = (c.rows.to(DEV), (ql.cumsum(0) - ql).int().to(DEV), (torch.tensor(c.lens) - ql).to(DEV), ql.to(DEV))
    got = kernels.paged_chunk_flash_attention_kv4(pad, c.pool.to(DEV), SCALE * LOG2E, tbl, *args, 5, table_kind="block")
    _within(got[:8], want, tol)
    # through the C entry, with and without a workspace: rows of no request keep what the output held
    lib, pool = _lib.lib(), c.pool.to(DEV)
    for ws_bytes in (0, lib.b200kv_kv4_chunk_workspace_bytes(2, 5, 8, 2, 128)):
        out = torch.full_like(pad, 9.0)
        ws = torch.zeros(max(1, ws_bytes), dtype=torch.uint8, device=DEV)
        rc = lib.b200kv_kv4_paged_prefill(
            pad.data_ptr(), pad.stride(0), pad.stride(1), pool.data_ptr(), pool.shape[0], pool.stride(0), tbl.data_ptr(),
            tbl.stride(0), 0, tbl.shape[0], tbl.shape[1], *(t.data_ptr() for t in args), 1, 2, pad.shape[0], 5, 8, 2, 128,
            16, SCALE * LOG2E, out.data_ptr(), out.stride(0), out.stride(1), ws.data_ptr() if ws_bytes else None, ws_bytes,
            kernels.status_tensor(0).data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        _within(out[:8], want, tol)
        assert bool((out[8:] == 9.0).all())
        assert not bool(ws[: kernels.DECODE_COUNTER_BYTES].any())


@pytest.mark.parametrize("special", [float("inf"), float("nan"), 60000.0])
def test_a_query_row_out_of_the_ordinary_stays_alone(special):
    c = Case(19, [90, 200, 31], 8, 2, [6, 6, 6])
    c.q[8, 3, 17] = special
    want, _, tol = c.want()
    assert int(want.isnan().any(-1).sum()) == (0 if math.isfinite(special) else 1)
    _within(c.prefill(), want, tol)
    d = Case(19, [90, 200, 31], 8, 2, [60, 130, 31])         # the tiles
    d.q[100, 3, 17] = special
    want, _, tol = d.want()
    _within(d.prefill(), want, tol)
    e = Case(19, [90, 200, 31], 8, 2)
    e.q[1, 3, 17] = special
    want, tol, _ = e.want()
    _within(e.decode(), want, tol)


@pytest.mark.parametrize("scale", [0.0, -SCALE, 30.0])
def test_decode_scales(scale):
    c = Case(23, [400, 3], 8, 2)
    want, tol, _ = c.want(scale)
    got = kernels.flash_decoding_kv4(c.q.to(DEV), c.pool.to(DEV), scale, c.tables("block"), torch.tensor(c.lens, device=DEV),
                                     400, b_req_idx=c.rows.to(DEV), table_kind="block")
    _within(got, want, tol)


def test_decode_out_may_be_q():
    c = Case(29, [3000, 40, 0, 700], 16, 2)
    want = c.decode().clone()
    q = c.q.to(DEV)
    out = kernels.flash_decoding_kv4(q, c.pool.to(DEV), SCALE, c.tables("block"), torch.tensor(c.lens, device=DEV), 3000,
                                     b_req_idx=c.rows.to(DEV), table_kind="block", out=q)
    assert out.data_ptr() == q.data_ptr() and torch.equal(out, want)


def test_largest_batches_and_refusals():
    kvh, b = 1, 4096
    rows = _randn(37, (64, 2, 128))
    pool = torch.zeros(4, 2, K4.BLOCK, dtype=torch.uint8)
    K4.append(rows, torch.arange(64, dtype=torch.int32), pool)
    values = K4.rows_of(pool, torch.arange(64))
    lens = torch.arange(b) % 60
    q = _randn(38, (60, 2, 128), 2)
    tbl = torch.arange(4, dtype=torch.int32).repeat(b, 1).to(DEV)
    dq, dpool = q[lens].to(DEV), pool.to(DEV)
    got = kernels.flash_decoding_kv4(dq, dpool, SCALE, tbl, lens.to(DEV), 64, table_kind="block").cpu()
    assert bool((got[lens == 0] == 0).all())
    want = torch.cat([K4.attention(q[n: n + 1], values[:n, :1], values[:n, 1:], n - 1, SCALE)[0] for n in range(60)])
    # 60 keys, values of at most 4.5 in magnitude: 2^-9 |v| of rounding in weights and output together, and 60 * 2^-24 * 5
    assert float((got.double() - want[lens]).abs().max()) <= 4.5 * 2 ** -9 + 60 * 5 * 2.0 ** -24
    ql = (lens > 0).long()
    chunk = kernels.paged_chunk_flash_attention_kv4(
        dq, dpool, SCALE * LOG2E, tbl, torch.arange(b, dtype=torch.int32, device=DEV), torch.arange(b, dtype=torch.int32, device=DEV),
        (lens - 1).clamp(min=0).to(DEV), ql.to(DEV), 1, table_kind="block").cpu()
    assert torch.equal(chunk[lens > 0], got[lens > 0])
    with pytest.raises(ValueError, match="decode shape"):      # a sequence too many
        kernels.flash_decoding_kv4(torch.zeros(b + 1, 2, 128, dtype=torch.float16, device=DEV), dpool, SCALE,
                                   tbl[:1].expand(1, 4), torch.ones(b + 1, dtype=torch.int32, device=DEV), 16,
                                   b_req_idx=torch.zeros(b + 1, dtype=torch.int32, device=DEV), table_kind="block")
    with pytest.raises(ValueError, match="decode shape"):      # 17 query heads to a KV head
        kernels.flash_decoding_kv4(torch.zeros(1, 17, 128, dtype=torch.float16, device=DEV), dpool, SCALE, tbl[:1],
                                   torch.ones(1, dtype=torch.int32, device=DEV), 16, table_kind="block")


def test_nothing_to_do():
    c = Case(43, [20], 4, 2)
    pool, tbl = c.pool.to(DEV), c.tables("block")
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert kernels.flash_decoding_kv4(torch.zeros(0, 4, 128, dtype=torch.float16, device=DEV), pool, SCALE, tbl,
                                      none, 0, b_req_idx=none, table_kind="block").shape == (0, 4, 128)
    assert kernels.paged_chunk_flash_attention_kv4(torch.zeros(0, 4, 128, dtype=torch.float16, device=DEV), pool, SCALE,
                                                   tbl, none, none, none, none, 0, table_kind="block").shape == (0, 4, 128)
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    out = kernels.flash_decoding_kv4(torch.ones(3, 4, 128, dtype=torch.float16, device=DEV), pool, SCALE, tbl, zero, 0,
                                     b_req_idx=zero, table_kind="block")
    assert bool((out == 0).all())
    kernels.paged_chunk_flash_attention_kv4(torch.ones(3, 4, 128, dtype=torch.float16, device=DEV), pool, SCALE, tbl,
                                            zero, zero, zero, zero, 4, table_kind="block")
    kernels.check_status(0)


def test_captured_steps_follow_lengths_tables_and_rows():
    """One captured decode and one captured chunk, replayed over other lengths, pages and requests."""
    cases = [Case(51, [2000, 40, 1], 8, 2, [4, 4, 1]), Case(52, [16, 1999, 300], 8, 2, [1, 2, 4]), Case(53, [5, 0, 31], 8, 2, [4, 0, 3])]
    pages, width = max(c.pool.shape[0] for c in cases), max(c.block.shape[1] for c in cases)
    pool = torch.zeros(pages, 4, K4.BLOCK, dtype=torch.uint8, device=DEV)
    tbl = torch.zeros(5, width, dtype=torch.int32, device=DEV)
    rows, lens, ctx, ql, start = (torch.zeros(3, dtype=torch.int32, device=DEV) for _ in range(5))
    q = torch.zeros(9, 8, 128, dtype=torch.float16, device=DEV)

    def step():
        return (kernels.flash_decoding_kv4(q[:3], pool, SCALE, tbl, lens, 2000, b_req_idx=rows, table_kind="block"),
                kernels.paged_chunk_flash_attention_kv4(q, pool, SCALE * LOG2E, tbl, rows, start, ctx, ql, 4, table_kind="block"))

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec, chunk = step()
    for c in cases + cases[::-1]:
        n = torch.tensor(c.q_lens, dtype=torch.int32)
        pool[: c.pool.shape[0]] = c.pool.to(DEV)
        tbl.zero_()
        tbl[:, : c.block.shape[1]] = c.block.to(DEV).clamp(max=pages - 1)
        rows.copy_(c.rows), lens.copy_(torch.tensor(c.lens)), ql.copy_(n), start.copy_(n.cumsum(0) - n)
        ctx.copy_(torch.tensor(c.lens) - n)
        q[: c.q.shape[0]] = c.q.to(DEV)
        g.replay()
        torch.cuda.synchronize()
        want, _, tol = c.want()
        _within(chunk[: c.q.shape[0]], want, tol)
        one = Case.__new__(Case)
        one.__dict__.update(c.__dict__)
        one.q, one.q_lens = q[:3].cpu(), [1, 1, 1]
        want, tol, _ = one.want()
        _within(dec, want, tol)
    kernels.check_status(0)


def test_branches_of_one_capture():
    """Two branches of a captured graph run at the same time: each has its own scratch."""
    a, b = Case(61, [3000, 40], 8, 1), Case(62, [2500, 700], 16, 2)
    want = a.decode().clone(), b.decode().clone()
    data = [(c.q.to(DEV), c.pool.to(DEV), SCALE, c.tables("block"), torch.tensor(c.lens, device=DEV), max(c.lens)) for c in (a, b)]
    rows = a.rows.to(DEV), b.rows.to(DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g, outs = torch.cuda.CUDAGraph(), ([], [])
    with torch.cuda.graph(g):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        for _ in range(4):
            outs[0].append(kernels.flash_decoding_kv4(*data[0], b_req_idx=rows[0], table_kind="block"))
        with torch.cuda.stream(side):
            for _ in range(4):
                outs[1].append(kernels.flash_decoding_kv4(*data[1], b_req_idx=rows[1], table_kind="block"))
        here.wait_stream(side)
    for _ in range(10):
        g.replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            for o in outs[i]:
                assert torch.equal(o, want[i])


FIRST_CALL = """
import sys, torch
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
from llama_lite_npu_b200 import kernels
from oracle import kv4_oracle as K4
import math
g0 = torch.Generator().manual_seed(1)
rows = torch.randn(40, 4, 128, generator=g0).half()
q = torch.randn(3, 8, 128, generator=g0).half()
pool = torch.zeros(3, 4, 1152, dtype=torch.uint8)
want_pool = pool.clone()
slots = torch.arange(40, dtype=torch.int32)
K4.append(rows, slots, want_pool)
d = lambda t: t.to("cuda:0")
drows, dq, dpool, dslots = d(rows), d(q), d(pool), d(slots)
tbl, lens, one = d(torch.arange(3, dtype=torch.int32).view(1, 3).repeat(3, 1)), d(torch.tensor([40, 17, 1])), d(torch.tensor([3]))
z = d(torch.zeros(1, dtype=torch.int32))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    kernels.update_kv_buffer_kv4(drows, dslots, dpool)
    back = kernels.gather_kv_buffer_kv4(dpool, dslots)
    dec = kernels.flash_decoding_kv4(dq, dpool, 1 / math.sqrt(128), tbl, lens, 48, table_kind="block")
    chunk = kernels.paged_chunk_flash_attention_kv4(dq, dpool, 1.4426950408889634 / math.sqrt(128), tbl, z, z, one + 31, one, 3, table_kind="block")
for _ in range(3):
    g.replay()
torch.cuda.synchronize()
assert torch.equal(dpool.cpu(), want_pool)
v = K4.rows_of(want_pool, slots)
assert torch.equal(back.cpu(), v.half())
for got, n, i in ((dec, 40, 0), (dec, 17, 1), (dec, 1, 2), (chunk, 35, 0), (chunk, 36, 1), (chunk, 37, 2)):
    want = K4.attention(q[i:i + 1], v[:n, :2], v[:n, 2:], n - 1, 1 / math.sqrt(128))[0][0]
    assert float((got[i].cpu().double() - want).abs().max()) < 4.5 * 2 ** -8, (n, i)
kernels.check_status(0)
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture(tmp_path):
    """Nothing was called before the capture: no workspace, no status word, no attribute set."""
    f = tmp_path / "first.py"
    f.write_text(FIRST_CALL.format(root=ROOT))
    r = subprocess.run([sys.executable, str(f)], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


def test_work_on_a_side_stream_follows_that_stream():
    """Inputs written on a side stream just before the call; the default stream takes no part."""
    c = Case(71, [600, 33], 8, 2, [3, 2])
    want, _, tol = c.want()
    side = torch.cuda.Stream()
    q, pool = torch.empty_like(c.q, device=DEV), torch.empty_like(c.pool, device=DEV)
    src_q, src_pool = c.q.to(DEV), c.pool.to(DEV)
    ql = torch.tensor(c.q_lens)
    args = (c.tables("block"), c.rows.to(DEV), (ql.cumsum(0) - ql).int().to(DEV), (torch.tensor(c.lens) - ql).to(DEV), ql.to(DEV))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(5):
            q.zero_(), pool.zero_()
            q.copy_(src_q), pool.copy_(src_pool)
            got = kernels.paged_chunk_flash_attention_kv4(q, pool, SCALE * LOG2E, *args, 3, table_kind="block")
            _within(got, want, tol)


def test_prefill_refuses_scales_that_are_not_positive():
    c = Case(81, [20], 4, 2, [20])
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises((ValueError, RuntimeError)):
            kernels.paged_chunk_flash_attention_kv4(
                c.q.to(DEV), c.pool.to(DEV), scale, c.tables("block"), c.rows.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV),
                torch.zeros(1, dtype=torch.int64, device=DEV), torch.tensor([20], device=DEV), 20, table_kind="block")


SPLIT = [   # few query tiles: their keys are cut into parts
    ([3000], [200], 2, 1), ([2500, 100], [130, 100], 16, 2), ([1700, 33, 600], [150, 33, 130], 3, 1), ([700], [300], 1, 1),
    ([2049], [129], 5, 1), ([513, 512], [257, 129], 1, 1), ([4000, 1], [140, 1], 8, 1), ([1300], [129], 8, 8),
]


@pytest.mark.parametrize("lens, q_lens, qh, kvh", SPLIT)
def test_keys_of_a_few_query_tiles_are_cut_into_parts(lens, q_lens, qh, kvh):
    c = Case(sum(lens) + qh, lens, qh, kvh, q_lens)
    want, _, tol = c.want()
    assert _lib.lib().b200kv_kv4_chunk_workspace_bytes(len(lens), max(q_lens), qh, kvh, 128) > 1 << 18
    got = c.prefill("block").clone()
    _within(got, want, tol)
    for _ in range(3):                        # the order in which parts arrive does not matter
        assert torch.equal(c.prefill("token", torch.int32), got)
    assert not any(bool(ws[: kernels.DECODE_COUNTER_BYTES].any()) for ws in kernels._kv4_workspace.values())


def test_cut_keys_nan_reaches_only_the_rows_that_see_it():
    c = Case(91, [2000, 800], 4, 2, [150, 130])
    x = _randn(92, (2000, 4, 128))
    x[1900, 2, 70] = float("nan")       # V of head 0, group 2, seen by rows 50 on
    x[1960, 1, 0] = float("inf")        # K of head 1
    x[1870, 3, 5] = float("-inf")       # V of head 1, group 0, seen by rows 20 on
    K4.append(x, c.slots[0], c.pool)
    c.values[0] = K4.rows_of(c.pool, c.slots[0])
    want, _, tol = c.want()
    got = c.prefill().cpu()
    assert bool(got[50:150, :2, 64:96].isnan().all()) and not bool(got[:50, :2].isnan().any())
    assert bool(got[110:150, 2:].isnan().all()) and bool(got[20:150, 2:, :32].isnan().all())
    assert not bool(got[:20].isnan().any()) and not bool(got[150:].isnan().any())
    _within(got, want, tol)


def test_cut_keys_value_ranges_and_unwritten_places():
    for gain_k, gain_v in ((15.0, 1.0), (1.0, 2000.0), (1.0, 1e-5)):
        c = Case(93, [1500, 31], 4, 1, [140, 31], gain_k=gain_k, gain_v=gain_v)
        want, _, tol = c.want()
        _within(c.prefill(), want, tol)
    fill = torch.full_like(c.pool, 0xF0)
    fill.view(torch.int16)[..., 512:] = GARBAGE[1]
    for s in c.slots:
        _take(fill, c.pool, s)
    _within(c.prefill(pool=fill.to(DEV)), want, tol)


def test_cut_keys_in_graphs_and_on_two_streams():
    a, b = Case(95, [3000], 8, 1, [200]), Case(96, [1500, 900], 4, 2, [130, 260])
    want = [c.prefill().clone() for c in (a, b)]
    calls = []
    for c in (a, b):
        ql = torch.tensor(c.q_lens)
        args = (c.q.to(DEV), c.pool.to(DEV), SCALE * LOG2E, c.tables("block"), c.rows.to(DEV), (ql.cumsum(0) - ql).int().to(DEV),
                (torch.tensor(c.lens) - ql).to(DEV), ql.to(DEV), max(c.q_lens))
        calls.append(lambda args=args: kernels.paged_chunk_flash_attention_kv4(*args, table_kind="block"))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for call in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([call() for _ in range(2)])
        graphs.append(g)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        eager = []
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
                eager.append(calls[i]())
        torch.cuda.synchronize()
        for i in (0, 1):
            for o in outs[i] + [eager[i]]:
                assert torch.equal(o, want[i])


@pytest.mark.parametrize("lens, q_lens, qh, kvh", [   # more than 128 columns, few heads and requests: streamed; the last two are not
    ([500], [40], 8, 1), ([300, 61], [60, 7], 4, 1), ([900], [128], 8, 1), ([77, 3], [32, 3], 16, 2), ([1000, 41, 5], [85, 30, 1], 4, 1),
    ([900], [129], 8, 1), ([400, 300], [65, 64], 8, 1)])
def test_chunks_of_many_columns_on_few_heads(lens, q_lens, qh, kvh):
    c = Case(sum(lens) + qh, lens, qh, kvh, q_lens)
    want, _, tol = c.want()
    _within(c.prefill("block"), want, tol)
    _within(c.prefill("token", torch.int32), want, tol)


def test_every_argument_may_be_junk():
    """Each argument of each operator replaced by objects of other kinds and tensors of other shapes: the call
    raises, keeps no reference and launches nothing."""
    c = Case(97, [20, 33], 4, 2, [1, 1])
    q, pool, tbl, rows = c.q.to(DEV), c.pool.to(DEV), c.tables("block"), c.rows.to(DEV)
    lens, one = torch.tensor(c.lens, device=DEV), torch.ones(2, dtype=torch.int64, device=DEV)
    start = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    kv, slots = _randn(98, (2, 4, 128)).to(DEV), torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    cs, w = torch.ones(2, 128, dtype=torch.float16, device=DEV), torch.ones(128, dtype=torch.float16, device=DEV)
    tensors = [q, pool, tbl, rows, lens, one, start, kv, slots, cs, w]
    before = [sys.getrefcount(t) for t in tensors]
    calls = [
        (kernels.update_kv_buffer_kv4, [kv, slots, pool], {}),
        (kernels.update_kv_buffer_kv4_split, [kv[:, :2], kv[:, 2:], slots, pool], {}),
        (kernels.fused_qk_norm_rope_append_kv4, [q, kv.flatten(1), w, w, 1e-6, cs, cs, slots, pool], {"out": torch.empty_like(q)}),
        (kernels.gather_kv_buffer_kv4, [pool, slots], {"out": torch.empty_like(kv)}),
        (kernels.flash_decoding_kv4, [q, pool, SCALE, tbl, lens, 33],
         {"b_req_idx": rows, "table_kind": "block", "page_size": 16, "out": torch.empty_like(q)}),
        (kernels.paged_chunk_flash_attention_kv4, [q, pool, SCALE, tbl, rows, start, lens - one, one, 1],
         {"table_kind": "block", "page_size": 16}),
    ]
    junk = [7, "junk", [1], object(), torch.zeros(3, 3, 3, 3, device=DEV), torch.zeros(0, device=DEV), torch.zeros(2, 2),
            torch.zeros(5, 128, dtype=torch.float16, device=DEV), torch.zeros((), device=DEV), torch.zeros(2, 4, 128, device=DEV)]
    raised = pytest.raises
    errors = (TypeError, ValueError, AttributeError, RuntimeError, IndexError)
    for fn, args, kw in calls:
        fn(*args, **kw)
        # numbers, and what may be left out, are looked at below
        for i, a in enumerate(args):
            for j in junk:
                if not isinstance(a, torch.Tensor) and isinstance(j, (int, torch.Tensor)):
                    continue
                with raised(errors):
                    fn(*args[:i], j, *args[i + 1:], **kw)
        for k, a in kw.items():
            for j in junk:
                if k == "page_size" and isinstance(j, (int, torch.Tensor)):
                    continue
                with raised(errors):
                    fn(*args, **{**kw, k: j})
    for bad in (1 << 40, -1, 1 << 70):
        with pytest.raises((ValueError, OverflowError)):
            kernels.flash_decoding_kv4(q, pool, SCALE, tbl, lens, 33, b_req_idx=rows, table_kind="block", page_size=bad)
        with pytest.raises((ValueError, OverflowError)):
            kernels.flash_decoding_kv4(q, pool, SCALE, tbl, lens, bad, b_req_idx=rows, table_kind="block")
    del calls, args, kw, a, j
    gc.collect()
    assert [sys.getrefcount(t) for t in tensors] == before
    torch.cuda.synchronize()
    kernels.check_status(0)


def test_tensors_of_a_device_that_is_not_current():
    """Every other answer about the current device is another one: each call is made again with the tensors' own."""
    c = Case(99, [40, 300], 4, 2, [1, 1])
    want, tol, tol_p = c.want()
    x = _randn(100, (2, 4, 128)).to(DEV)
    slots = torch.tensor([int(s[3]) for s in c.slots], dtype=torch.int32, device=DEV)
    cs = torch.ones(2, 128, dtype=torch.float16, device=DEV)
    plain = [c.pool.to(DEV) for _ in (0, 1)]
    kernels.update_kv_buffer_kv4(x, slots, plain[0])
    q_plain = kernels.fused_qk_norm_rope_append_kv4(c.q.to(DEV), x.flatten(1), None, None, 1e-6, cs, cs, slots, plain[1])
    asked = []
    parts = kernels._kv4_parts()
    parts["current_device"] = lambda: asked.append(0) or len(asked) % 2
    kernels._kv4.setup(parts)
    try:
        _within(c.decode(), want, tol)
        _within(c.prefill(), want, tol_p)
        pools = [c.pool.to(DEV) for _ in (0, 1)]
        kernels.update_kv_buffer_kv4(x, slots, pools[0])
        q = kernels.fused_qk_norm_rope_append_kv4(c.q.to(DEV), x.flatten(1), None, None, 1e-6, cs, cs, slots, pools[1])
        rows = kernels.gather_kv_buffer_kv4(pools[0], slots)
    finally:
        kernels._kv4.setup(kernels._kv4_parts())
    assert len(asked) == 10
    assert torch.equal(pools[0], plain[0]) and torch.equal(pools[1], plain[1]) and torch.equal(q, q_plain)
    assert torch.equal(rows.cpu(), K4.rows_of(plain[0].cpu(), slots.cpu()).half())


def test_counters_are_cleared_after_a_wait_that_ran_out():
    """A reported time-out clears the scratch of every shape that was in use, a larger shape's and the smaller one's."""
    a, b = Case(131, [3000, 40], 8, 1), Case(132, [400] * 9, 16, 4)
    want = [c.decode().clone() for c in (a, b, a)][1:]
    for ws in kernels._kv4_workspace.values():
        ws[: kernels.DECODE_COUNTER_BYTES] = 1
    kernels.status_tensor(0).fill_(104)
    with pytest.raises(RuntimeError, match="104"):
        kernels.check_status(0)
    assert not any(bool(ws[: kernels.DECODE_COUNTER_BYTES].any()) for ws in kernels._kv4_workspace.values())
    for _ in range(2):
        assert torch.equal(b.decode(), want[0]) and torch.equal(a.decode(), want[1])


def test_many_shapes_on_many_streams():
    """More shapes and streams than scratch is remembered for, in turn."""
    cases = [Case(140 + i, [50 * i + 5, 700 - 90 * i], 4 * (1 + i % 3), 1 + i % 2) for i in range(7)]
    want = [c.decode().clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for r in range(3):
        outs = []
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[(i + r) % 3]):
                outs.append(c.decode())
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)

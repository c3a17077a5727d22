"""The 4-bit paged cache on the GPU against its 64-bit statement (oracle/kv4_oracle.py).

Appends are held to the exact bytes, read-backs to the exactly rounded values.  Attention outputs are
held element by element to an error that is counted from the kernels' roundings (u = 2^-11, half a step of
fp16, relative):

* the output is rounded once:                                      u |o|
* a weight p is rounded to fp16 once (prefill) or twice, before and after it meets V's scale
  (decode), and prefill rounds V too:                              2 u sum p|v|
* prefill rounds K to fp16, so a score moves by at most u * dot with dot = scale * sum |q k| and a weight by
  twice that (itself and the sum it is divided by):                2 u dot sum p|v|
* 32-bit sums and the exponential: scores are sums of 128 products in 32 bits with at most 2^-20
  relative to dot, the exponential and the sums over keys 2^-18:   (2^-18 + 2 * 2^-20 dot) sum p|v|
* weights under 2^-14 of the largest lose bits in fp16, at most 2^-25 each before V's scale and,
  scaled, as much again:                                           keys * 2^-24 max|v|
"""

import math

import pytest
import torch

from llama_lite_npu_b200 import _lib, kernels, workloads as W
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 1.0 / math.sqrt(128)
LOG2E = 1.4426950408889634
U = 2.0 ** -11


@pytest.fixture(scope="module", autouse=True)
def _lib_loaded(built_lib):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    yield
    kernels.check_status(0)


def _randn(seed, shape, stream=1, gain=1.0):
    return (W.hash_normal_fp16(seed, shape, stream).float() * gain).half()


def _slots(seed, n, total):
    return torch.from_numpy(W.hash_permutation(seed, total, 9)[:n].astype("int32"))


def _noise_pool(seed, pages, kvh):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 256, (pages, 2 * kvh, K4.BLOCK), dtype=torch.uint8, generator=g)


# ---------------------------------------------------------------------------------------------
# append and read-back
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n, kvh, gain", [(1, 1, 1.0), (3, 8, 1.0), (4, 2, 1e-4), (5, 1, 2e-7), (37, 5, 900.0), (130, 4, 1.0)])
def test_append_writes_the_exact_bytes(n, kvh, gain):
    x = _randn(n, (n, 2 * kvh, 128), 1, gain)
    x[0, 0, :4] = torch.tensor([0.5, 3.5, -3.5, 7.0]).half()       # borders of the codes when the scale is 1
    x[0, 0, 4:32] = 0
    pool = _noise_pool(n, 12, kvh)
    slots = _slots(n, n, 12 * 16)
    want = pool.clone()
    K4.append(x, slots, want)
    dpool = pool.to(DEV)
    kernels.update_kv_buffer_kv4(x.to(DEV), slots.to(DEV), dpool)
    assert torch.equal(dpool.cpu(), want)
    split = pool.to(DEV)
    kernels.update_kv_buffer_kv4_split(x[:, :kvh].contiguous().to(DEV), x[:, kvh:].to(DEV), slots.to(DEV), split)
    assert torch.equal(split.cpu(), want)
    back = kernels.gather_kv_buffer_kv4(dpool, slots.to(DEV))
    assert torch.equal(back.cpu(), K4.rows_of(want, slots).half())


def test_append_every_fp16_magnitude():
    """A row per exponent of fp16, subnormals, the largest value, ties at every code border."""
    rows = []
    for e in range(-24, 16):
        row = _randn(100 + e, (128,), 1, 1.0).float() * 2.0 ** e / 8
        row[:15] = torch.arange(-7, 8).float() * 2.0 ** e / 8
        row[32:47] = (torch.arange(-7, 8).float() + 0.5) * 2.0 ** e / 8
        row[47] = 7 * 2.0 ** e / 8
        rows.append(row.clamp(-65504, 65504).half())
    x = torch.stack(rows).unsqueeze(1).repeat(1, 2, 1).contiguous()
    n = x.shape[0]
    pool = torch.zeros(3, 2, K4.BLOCK, dtype=torch.uint8)
    slots = _slots(5, n, 48)
    want = pool.clone()
    K4.append(x, slots, want)
    dpool = pool.to(DEV)
    kernels.update_kv_buffer_kv4(x.to(DEV), slots.to(DEV), dpool)
    assert torch.equal(dpool.cpu(), want)


def test_append_non_finite_groups_read_back_as_nan():
    x = _randn(9, (3, 2, 128))
    x[0, 0, 5], x[1, 1, 64], x[2, 0, 127] = float("inf"), float("nan"), float("-inf")
    slots = torch.tensor([17, 2, 30], dtype=torch.int32)
    pool = torch.zeros(2, 2, K4.BLOCK, dtype=torch.uint8, device=DEV)
    kernels.update_kv_buffer_kv4(x.to(DEV), slots.to(DEV), pool)
    want = torch.zeros(2, 2, K4.BLOCK, dtype=torch.uint8)
    K4.append(x, slots, want)
    got = kernels.gather_kv_buffer_kv4(pool, slots.to(DEV)).cpu().float()
    ref = K4.rows_of(want, slots).half().float()
    assert torch.equal(got.isnan(), ref.isnan()) and int(got.isnan().sum()) == 96
    assert torch.equal(got.nan_to_num(0), ref.nan_to_num(0))


def test_append_bad_slots_strides_and_views():
    n, kvh = 21, 3
    wide = _randn(7, (n, 2 * kvh * 128 + 40)).to(DEV)
    x = wide[:, : 2 * kvh * 128].view(n, 2 * kvh, 128)                # token stride larger than a row
    big = _noise_pool(7, 9, kvh + 1).to(DEV)
    store = torch.zeros(9, 2 * kvh * K4.BLOCK + 64, dtype=torch.uint8, device=DEV)
    pool = store[:, : 2 * kvh * K4.BLOCK].view(9, 2 * kvh, K4.BLOCK)  # page stride larger than a page
    slots = _slots(7, n, 9 * 16)
    slots[4], slots[9] = -1, 9 * 16
    every_other = torch.stack((slots, slots), 1).to(DEV)[:, 0]        # a strided index tensor
    kernels.update_kv_buffer_kv4(x, every_other, pool)
    with pytest.raises(RuntimeError, match="slot_mapping"):
        kernels.check_status(0)
    want = torch.zeros(9, 2 * kvh, K4.BLOCK, dtype=torch.uint8)
    K4.append(x.cpu(), slots, want)
    assert torch.equal(pool.cpu(), want)
    assert bool((store[:, 2 * kvh * K4.BLOCK:] == 0).all())
    out = torch.full((n, 2 * kvh + 1, 128), 3.0, dtype=torch.float16, device=DEV)
    got = kernels.gather_kv_buffer_kv4(pool, slots.to(DEV), out=out[:, : 2 * kvh])
    with pytest.raises(RuntimeError, match="slot_mapping"):
        kernels.check_status(0)
    ok = (slots >= 0) & (slots < 9 * 16)
    assert torch.equal(got.cpu()[ok], K4.rows_of(want, slots[ok]).half())
    assert bool((got.cpu()[~ok] == 0).all()) and bool((out[:, 2 * kvh:] == 3.0).all())
    assert big.shape[1] == 2 * (kvh + 1)
    with pytest.raises(ValueError):
        kernels.update_kv_buffer_kv4(x, slots.to(DEV), big)           # another number of heads
    # nothing to do
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    kernels.update_kv_buffer_kv4(x[:0], none, pool)
    assert kernels.gather_kv_buffer_kv4(pool, none).shape == (0, 2 * kvh, 128)


@pytest.mark.parametrize("n, qh, kvh, norm, half_cos", [(1, 1, 1, True, False), (6, 16, 8, True, True), (41, 10, 2, False, False),
                                                       (129, 8, 4, True, False)])
def test_fused_norm_rope_append(n, qh, kvh, norm, half_cos):
    fused = _randn(n, (n, (qh + 2 * kvh) * 128 + 16)).to(DEV)
    xq = fused[:, : qh * 128].view(n, qh, 128)
    xkv = fused[:, qh * 128: (qh + 2 * kvh) * 128]
    wq = (1 + 0.3 * _randn(n, (128,), 2).float()).half() if norm else None
    wk = (1 + 0.3 * _randn(n, (128,), 3).float()).half() if norm else None
    ang = 3.0 * _randn(n, (n, 64), 4).float()
    cos, sin = ang.cos().half(), ang.sin().half()
    if not half_cos:
        cos, sin = torch.cat((cos, cos), 1), torch.cat((sin, sin), 1)
    slots = _slots(n, n, 11 * 16)
    pool = _noise_pool(n, 11, kvh)
    q0, kv0 = xq.cpu(), xkv.cpu().view(n, 2 * kvh, 128)
    c2, s2 = (torch.cat((t, t), 1) if t.shape[1] == 64 else t for t in (cos, sin))
    want = pool.clone()
    K4.append(torch.cat((K4.norm_rope(kv0[:, :kvh], wk, 1e-6, c2, s2), kv0[:, kvh:]), 1), slots, want)
    up = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    dpool, out = pool.to(DEV), torch.empty(n, qh, 128, dtype=torch.float16, device=DEV)
    got = kernels.fused_qk_norm_rope_append_kv4(xq, xkv, up(wq), up(wk), 1e-6, up(cos), up(sin), up(slots), dpool, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(xq.cpu(), q0)
    assert torch.equal(dpool.cpu(), want)
    # Q: 32-bit statistics may move x * rrms across one rounding to fp16 (a whole step, 2^-10), the
    # product with the weight is rounded (2^-11 against the statement's own 2^-11), then the rotation's
    # rounding: each element is within 4 half steps of the terms it is a sum of
    exact = K4.norm_rope(q0, wq, 1e-6, c2, s2, round_last=False)
    y = K4.norm_rope(q0, wq, 1e-6, torch.ones_like(c2), torch.zeros_like(s2), round_last=False).abs()
    terms = torch.cat((y[..., :64] * c2[:, None, :64].double().abs() + y[..., 64:] * s2[:, None, :64].double().abs(),
                       y[..., 64:] * c2[:, None, :64].double().abs() + y[..., :64] * s2[:, None, :64].double().abs()), -1)
    assert bool(((got.cpu().double() - exact).abs() <= 4 * U * terms + U * exact.abs() + 2.0 ** -24).all())
    # in place
    again = fused.clone()
    xq2, xkv2 = again[:, : qh * 128].view(n, qh, 128), again[:, qh * 128: (qh + 2 * kvh) * 128]
    dpool2 = pool.to(DEV)
    kernels.fused_qk_norm_rope_append_kv4(xq2, xkv2, up(wq), up(wk), 1e-6, up(cos), up(sin), up(slots), dpool2)
    assert torch.equal(xq2, got) and torch.equal(dpool2, dpool)
    assert torch.equal(again[:, qh * 128:], fused[:, qh * 128:])


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
class Case:
    """A 4-bit pool with sequences on shuffled pages; table rows in another order than the batch."""

    def __init__(self, seed, lens, qh, kvh, q_lens=None, gain_k=1.0, gain_v=1.0, noise=True):
        self.lens, self.qh, self.kvh = list(lens), qh, kvh
        b = len(self.lens)
        self.q_lens = [1] * b if q_lens is None else list(q_lens)
        pages = [(n + 15) // 16 for n in self.lens]
        total = sum(pages) + 3
        width = max(pages + [1]) + 1
        order = torch.from_numpy(W.hash_permutation(seed, total, 3))
        self.rows = torch.from_numpy(W.hash_permutation(seed, b + 2, 4)[:b].astype("int32"))
        self.block = torch.full((b + 2, width), 1 << 29, dtype=torch.int32)    # unused entries name no page
        at = 0
        for i, np_ in enumerate(pages):
            self.block[int(self.rows[i]), :np_] = order[at: at + np_].int()
            at += np_
        self.token = (self.block.unsqueeze(-1) * 16 + torch.arange(16, dtype=torch.int32)).flatten(1).contiguous()
        self.pool = _noise_pool(seed, total, kvh) if noise else torch.zeros(total, 2 * kvh, K4.BLOCK, dtype=torch.uint8)
        if noise:        # NaN scales in every place that is never written
            self.pool.view(torch.float16)[..., 512:] = float("nan")
        self.slots = [self.token[int(self.rows[i]), :n] for i, n in enumerate(self.lens)]
        self.values = []
        for i, n in enumerate(self.lens):
            x = _randn(seed * 31 + i, (n, 2 * kvh, 128), 5).float()
            x[:, :kvh] *= gain_k
            x[:, kvh:] *= gain_v
            K4.append(x.half(), self.slots[i], self.pool)
            self.values.append(K4.rows_of(self.pool, self.slots[i]))
        self.q = _randn(seed, (sum(self.q_lens), qh, 128), 6)

    def tables(self, kind):
        return (self.token if kind == "token" else self.block).to(DEV)

    def want(self, scale=SCALE):
        outs, tols_dec, tols_pre = [], [], []
        begin = 0
        for i, n in enumerate(self.lens):
            m = self.q_lens[i]
            k, v = self.values[i][:, : self.kvh], self.values[i][:, self.kvh:]
            o, mag, dot = K4.attention(self.q[begin: begin + m], k, v, n - m, scale)
            vmax = v.nan_to_num(0.0).abs().max() if n else torch.tensor(0.0)
            base = U * o.abs() + 2.0 ** -25 + (2 * U + 2.0 ** -18 + 2.0 ** -19 * dot) * mag + n * 2.0 ** -24 * vmax
            outs.append(o)
            tols_dec.append(base)
            tols_pre.append(base + 2 * U * dot * mag)
            begin += m
        return torch.cat(outs), torch.cat(tols_dec), torch.cat(tols_pre)

    def decode(self, kind="block", lens_dtype=torch.int64, **kw):
        lens = torch.tensor(self.lens, dtype=lens_dtype, device=DEV)
        return kernels.flash_decoding_kv4(self.q.to(DEV), self.pool.to(DEV), SCALE, self.tables(kind), lens,
                                          max(self.lens + [0]), b_req_idx=self.rows.to(DEV), table_kind=kind, **kw)

    def prefill(self, kind="block", lens_dtype=torch.int64, pool=None):
        ql = torch.tensor(self.q_lens, dtype=lens_dtype)
        start = (ql.cumsum(0) - ql).int()
        ctx = torch.tensor(self.lens, dtype=lens_dtype) - ql
        return kernels.paged_chunk_flash_attention_kv4(
            self.q.to(DEV), self.pool.to(DEV) if pool is None else pool, SCALE * LOG2E, self.tables(kind),
            self.rows.to(DEV), start.to(DEV), ctx.to(lens_dtype).to(DEV), ql.to(DEV), max(self.q_lens), table_kind=kind)


def _within(got, want, tol):
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    off = ((got - want).abs() - tol).nan_to_num(-1.0)
    assert float(off.max()) <= 0, f"worst excess {float(off.max()):.3e} at {int(off.argmax())}"


DECODE = [
    ([1], 1, 1), ([0], 4, 2), ([0, 0, 5], 8, 1), ([16, 17, 15, 1, 0, 33], 16, 2), ([300, 1, 64], 5, 1),
    ([700], 32, 2), ([40, 900, 3], 12, 1), ([2100, 77], 8, 8), ([129] * 9, 24, 3), ([63, 64, 65] * 5, 7, 1),
    ([5000], 16, 1),
]


@pytest.mark.parametrize("lens, qh, kvh", DECODE)
def test_decode(lens, qh, kvh):
    c = Case(len(lens) * 1000 + sum(lens), lens, qh, kvh)
    want, tol, _ = c.want()
    _within(c.decode("block"), want, tol)
    _within(c.decode("token", torch.int32, metadata_fresh=True), want, tol)


@pytest.mark.parametrize("gain_k, gain_v", [(1.0, 1e-6), (1.0, 3e-4), (1.0, 3000.0), (12.0, 1.0), (0.0, 1.0), (1.0, 0.0)])
def test_decode_value_ranges(gain_k, gain_v):
    c = Case(77, [517, 30], 8, 2, gain_k=gain_k, gain_v=gain_v)
    want, tol, _ = c.want()
    _within(c.decode(), want, tol)


def test_decode_v_scales_far_apart():
    """The token with nearly all the weight has small values, others a thousand times larger ones."""
    c = Case(5, [400], 4, 1)
    x = _randn(6, (400, 2, 128)).float()
    x[:, 1] *= torch.where(torch.arange(400) % 7 == 0, 1000.0, 1.0).unsqueeze(-1)
    x[123, 0] = 6 * c.q[0, 0].float()
    x[123, 1] *= 0.01
    K4.append(x.half(), c.slots[0], c.pool)
    c.values[0] = K4.rows_of(c.pool, c.slots[0])
    want, tol, _ = c.want()
    _within(c.decode(), want, tol)


def test_decode_long_split_sequences_and_many_short_ones():
    lens = [9000, 2, 0, 1] + [20] * 150 + [3000]         # more sequences in a team than its cache of lengths
    c = Case(11, lens, 4, 1)
    want, tol, _ = c.want()
    _within(c.decode(), want, tol)


def test_decode_nan_and_infinity_stay_with_their_sequence():
    c = Case(21, [50, 60, 70], 8, 2)
    x = _randn(22, (60, 4, 128))
    x[10, 0, 5] = float("inf")          # K of head 0
    x[11, 3, 40] = float("nan")         # V of head 1, one group
    K4.append(x, c.slots[1], c.pool)
    c.values[1] = K4.rows_of(c.pool, c.slots[1])
    got = c.decode().cpu()
    want, tol, _ = c.want()
    assert not bool(got[0].isnan().any()) and not bool(got[2].isnan().any())
    assert bool(got[1, :4].isnan().all())
    assert bool(got[1, 4:, 32:64].isnan().all()) and not bool(got[1, 4:, :32].isnan().any())
    _within(got[[0, 2]], want[[0, 2]], tol[[0, 2]])


def test_decode_strided_q_and_out_and_zero_rows():
    c = Case(31, [0, 45, 0], 6, 2)
    want, tol, _ = c.want()
    buf = torch.full((3, 8, 128), 5.0, dtype=torch.float16, device=DEV)
    qbuf = torch.zeros(3, 10, 128, dtype=torch.float16, device=DEV)
    qbuf[:, 2:8] = c.q.to(DEV)
    out = kernels.flash_decoding_kv4(qbuf[:, 2:8], c.pool.to(DEV), SCALE, c.tables("block"),
                                     torch.tensor(c.lens, device=DEV), 45, b_req_idx=c.rows.to(DEV), table_kind="block",
                                     out=buf[:, 1:7])
    _within(out, want, tol)
    assert bool((out[[0, 2]] == 0).all()) and bool((buf[:, 0] == 5).all()) and bool((buf[:, 7] == 5).all())


def test_decode_bad_pages_rows_and_lengths_are_reported():
    c = Case(41, [100, 100, 100], 8, 1)
    want, tol, _ = c.want()
    tbl = c.block.clone()
    tbl[int(c.rows[1]), 2] = c.pool.shape[0]                  # one past the pool
    lens = torch.tensor([100, 100, 100], device=DEV)
    got = kernels.flash_decoding_kv4(c.q.to(DEV), c.pool.to(DEV), SCALE, tbl.to(DEV), lens, 100,
                                     b_req_idx=c.rows.to(DEV), table_kind="block")
    with pytest.raises(RuntimeError, match="page/token table"):
        kernels.check_status(0)
    _within(got[[0, 2]], want[[0, 2]], tol[[0, 2]])
    tok = c.token.clone()
    tok[int(c.rows[1]), 16] += 3                               # a page may not start inside a page
    got = kernels.flash_decoding_kv4(c.q.to(DEV), c.pool.to(DEV), SCALE, tok.to(DEV), lens, 100,
                                     b_req_idx=c.rows.to(DEV), table_kind="token")
    with pytest.raises(RuntimeError, match="page/token table"):
        kernels.check_status(0)
    _within(got[[0, 2]], want[[0, 2]], tol[[0, 2]])
    rows = c.rows.clone()
    rows[1] = 99                                               # a request the table does not have: an empty sequence
    got = kernels.flash_decoding_kv4(c.q.to(DEV), c.pool.to(DEV), SCALE, c.tables("block"), lens, 100,
                                     b_req_idx=rows.to(DEV), table_kind="block")
    with pytest.raises(RuntimeError, match="length"):
        kernels.check_status(0)
    _within(got[[0, 2]], want[[0, 2]], tol[[0, 2]])
    assert bool((got[1] == 0).all())


PREFILL = [
    ([1], [1], 1, 1), ([5, 9], [5, 2], 4, 2), ([40, 16, 17], [40, 1, 17], 6, 2), ([300, 130], [200, 130], 8, 1),
    ([700, 33, 129], [3, 33, 128], 16, 2), ([260], [260], 3, 3), ([1000, 90], [130, 4], 16, 1),
]


@pytest.mark.parametrize("lens, q_lens, qh, kvh", PREFILL)
def test_prefill(lens, q_lens, qh, kvh):
    c = Case(sum(lens), lens, qh, kvh, q_lens)
    want, _, tol = c.want()
    _within(c.prefill("block"), want, tol)
    _within(c.prefill("token", torch.int32), want, tol)


def test_prefill_value_ranges():
    for gain_v in (1e-5, 800.0):
        c = Case(55, [200, 90], 4, 2, [60, 90], gain_v=gain_v)
        want, _, tol = c.want()
        _within(c.prefill(), want, tol)


def test_prefill_nan_reaches_only_the_rows_that_see_it():
    c = Case(61, [150, 150], 4, 2, [150, 20])
    x = _randn(62, (150, 4, 128))
    x[100, 2, 70] = float("nan")        # V of head 0, group 2, at position 100
    x[120, 1, 0] = float("inf")         # K of head 1 at position 120
    K4.append(x, c.slots[0], c.pool)
    c.values[0] = K4.rows_of(c.pool, c.slots[0])
    want, _, tol = c.want()
    got = c.prefill().cpu()
    assert not bool(got[:100].isnan().any()) and not bool(got[150:].isnan().any())
    assert bool(got[100:150, :2, 64:96].isnan().all()) and not bool(got[100:120, :, :64].isnan().any())
    assert bool(got[120:150, 2:].isnan().all())
    _within(got, want, tol)


CHUNK = [   # at most 128 columns (query rows x heads of a group): streamed like a decode step
    ([40], [1], 8, 1), ([33, 17, 500], [7, 7, 7], 8, 1), ([64, 1, 2000], [4, 1, 2], 16, 1), ([300, 5], [5, 5], 3, 3),
    ([129, 700], [16, 3], 8, 2), ([90, 1500, 31], [2, 8, 8], 64, 8), ([200, 100], [3, 0], 20, 2), ([4000], [6], 10, 1),
    ([21, 22, 23, 24] * 40, [1, 2, 3, 4] * 40, 4, 1), ([64], [64], 1, 1),
]


@pytest.mark.parametrize("lens, q_lens, qh, kvh", CHUNK)
def test_short_chunks(lens, q_lens, qh, kvh):
    c = Case(sum(lens) + len(lens), lens, qh, kvh, q_lens)
    want, _, tol = c.want()
    pool = c.pool.to(DEV)
    got = c.prefill("block", pool=pool)
    _within(got, want, tol)
    _within(c.prefill("token", torch.int32), want, tol)
    # without a workspace the same call goes through the tensor-core tiles
    lib, ql = _lib.lib(), torch.tensor(c.q_lens)
    q, tbl, rows = c.q.to(DEV), c.tables("block"), c.rows.to(DEV)
    start, ctx, qd = (ql.cumsum(0) - ql).int().to(DEV), (torch.tensor(c.lens) - ql).to(DEV), ql.to(DEV)
    out = torch.zeros_like(q)
    need = lib.b200kv_kv4_chunk_workspace_bytes(len(lens), max(q_lens), qh, kvh, 128)
    assert need > 0
    args = (q.data_ptr(), q.stride(0), q.stride(1), pool.data_ptr(), pool.shape[0], pool.stride(0), tbl.data_ptr(),
            tbl.stride(0), 0, tbl.shape[0], tbl.shape[1], rows.data_ptr(), start.data_ptr(), ctx.data_ptr(),
            qd.data_ptr(), 1, len(lens), q.shape[0], max(q_lens), qh, kvh, 128, 16, SCALE * LOG2E, out.data_ptr(),
            out.stride(0), out.stride(1))
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.b200kv_kv4_paged_prefill(*args, 0, 0, kernels.status_tensor(0).data_ptr(), stream) == 0
    _within(out, want, tol)
    # and one that is too small is refused
    assert lib.b200kv_kv4_paged_prefill(*args, pool.data_ptr(), need - 1, None, stream) == 4


def test_short_chunk_nan_reaches_only_the_rows_that_see_it():
    c = Case(63, [150, 90], 8, 2, [8, 8])
    x = _randn(64, (150, 4, 128))
    x[146, 2, 70] = float("nan")        # V of head 0, group 2, at the chunk's row 4
    x[148, 1, 0] = float("inf")         # K of head 1 at row 6
    K4.append(x, c.slots[0], c.pool)
    c.values[0] = K4.rows_of(c.pool, c.slots[0])
    want, _, tol = c.want()
    got = c.prefill().cpu()
    assert not bool(got[:4].isnan().any()) and not bool(got[8:].isnan().any())
    assert bool(got[4:8, :4, 64:96].isnan().all()) and not bool(got[4:6, :, :64].isnan().any())
    assert bool(got[6:8, 4:].isnan().all())
    _within(got, want, tol)


@pytest.mark.parametrize("max_q", [4, 200])
def test_a_chunk_longer_than_stated_is_skipped(max_q):
    c = Case(65, [300, 300], 8, 1, [max_q // 2, max_q + 1])
    want, _, tol = c.want()
    ql = torch.tensor(c.q_lens)
    got = kernels.paged_chunk_flash_attention_kv4(
        c.q.to(DEV), c.pool.to(DEV), SCALE * LOG2E, c.tables("block"), c.rows.to(DEV), (ql.cumsum(0) - ql).int().to(DEV),
        (torch.tensor(c.lens) - ql).to(DEV), ql.to(DEV), max_q, table_kind="block")
    with pytest.raises(RuntimeError, match="length"):
        kernels.check_status(0)
    _within(got[: max_q // 2], want[: max_q // 2], tol[: max_q // 2])


def test_prefill_skips_a_request_the_table_cannot_hold():
    c = Case(71, [64, 80], 4, 1, [64, 10])
    want, _, tol = c.want()
    rows = c.rows.clone()
    rows[0] = 50
    ql = torch.tensor(c.q_lens)
    got = kernels.paged_chunk_flash_attention_kv4(
        c.q.to(DEV), c.pool.to(DEV), SCALE * LOG2E, c.tables("block"), rows.to(DEV), torch.tensor([0, 64], dtype=torch.int32).to(DEV),
        torch.tensor([0, 70]).to(DEV), ql.to(DEV), 64, table_kind="block")
    with pytest.raises(RuntimeError, match="length"):
        kernels.check_status(0)
    _within(got[64:], want[64:], tol[64:])


# ---------------------------------------------------------------------------------------------
# refusals in Python, streams, graphs
# ---------------------------------------------------------------------------------------------
def test_python_refusals():
    c = Case(81, [20, 20], 4, 2)
    q, pool, tbl = c.q.to(DEV), c.pool.to(DEV), c.tables("block")
    lens, rows = torch.tensor(c.lens, device=DEV), c.rows.to(DEV)
    call = lambda **kw: kernels.flash_decoding_kv4(  # noqa: E731
        kw.pop("q", q), kw.pop("pool", pool), SCALE, kw.pop("tbl", tbl), kw.pop("lens", lens), kw.pop("max_len", 20),
        b_req_idx=kw.pop("rows", rows), table_kind=kw.pop("kind", "block"), **kw)
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q.cpu()), dict(pool=pool.short()), dict(pool=pool[:, :3]),
                dict(pool=pool[:, :, :1000]), dict(pool=pool[:0]), dict(tbl=tbl.long()), dict(tbl=tbl.cpu()),
                dict(lens=lens[:1]), dict(lens=lens.float()), dict(rows=rows.long()), dict(max_len=10 ** 6),
                dict(kind="dense"), dict(kind="what"), dict(out=q.float()), dict(page_size=32), dict(lens=lens.cpu())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError):
        kernels.gather_kv_buffer_kv4(pool, torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):
        kernels.update_kv_buffer_kv4(torch.zeros(1, 4, 128, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), pool)
    torch.cuda.synchronize()
    kernels.check_status(0)


def test_debug_mode_refuses_before_launch():
    c = Case(91, [20], 4, 2)
    pool = c.pool.to(DEV)
    x = _randn(92, (2, 4, 128)).to(DEV)
    kernels.set_debug(True)
    try:
        with pytest.raises(ValueError, match="outside the pool"):
            kernels.update_kv_buffer_kv4(x, torch.tensor([1, 10 ** 6], dtype=torch.int32, device=DEV), pool)
        with pytest.raises(ValueError, match="different K/V rows"):
            kernels.update_kv_buffer_kv4(x, torch.tensor([5, 5], dtype=torch.int32, device=DEV), pool)
        with pytest.raises(ValueError, match="length"):
            kernels.flash_decoding_kv4(c.q.to(DEV), pool, SCALE, c.tables("block"), torch.tensor([20], device=DEV), 10,
                                       b_req_idx=c.rows.to(DEV), table_kind="block")
    finally:
        kernels.set_debug(False)
    assert torch.equal(pool.cpu(), c.pool)


def test_two_streams_at_once_and_repeated_calls_agree():
    a, b = Case(101, [3000, 40], 8, 1), Case(102, [2500, 700], 16, 2)
    first = a.decode().clone(), b.decode().clone()
    args = []
    for c in (a, b):
        args.append((c.q.to(DEV), c.pool.to(DEV), SCALE, c.tables("block"), torch.tensor(c.lens, device=DEV), max(c.lens)))
    rows = a.rows.to(DEV), b.rows.to(DEV)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = ([], [])
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                outs[i].append(kernels.flash_decoding_kv4(*args[i], b_req_idx=rows[i], table_kind="block"))
    torch.cuda.synchronize()
    for i in (0, 1):
        for o in outs[i]:
            assert torch.equal(o, first[i])


def test_two_graphs_replayed_side_by_side():
    """Each captured graph has a workspace of its own, so replays on two streams and eager calls may overlap."""
    a, b = Case(111, [4000, 40], 8, 1), Case(112, [2500, 700], 16, 2)
    want = a.decode().clone(), b.decode().clone()
    data = [(c.q.to(DEV), c.pool.to(DEV), SCALE, c.tables("block"), torch.tensor(c.lens, device=DEV), max(c.lens)) for c in (a, b)]
    rows = a.rows.to(DEV), b.rows.to(DEV)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = [kernels.flash_decoding_kv4(*data[i], b_req_idx=rows[i], table_kind="block") for _ in range(3)]
        graphs.append(g)
        outs.append(o)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        eager = kernels.flash_decoding_kv4(*data[0], b_req_idx=rows[0], table_kind="block")
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for i in (0, 1):
            for o in outs[i]:
                assert torch.equal(o, want[i])


def test_append_then_decode_on_the_same_stream_sees_the_new_rows():
    """append -> decode back to back, eagerly and as a graph: the decode's early start must not read old rows."""
    c = Case(121, [33, 500, 16], 8, 2)
    pool = c.pool.to(DEV)
    new = [_randn(130 + s, (3, 4, 128)) for s in range(4)]
    slots = torch.tensor([int(s[-1]) for s in c.slots], dtype=torch.int32)
    dslots, tbl, rows, lens = slots.to(DEV), c.tables("block"), c.rows.to(DEV), torch.tensor(c.lens, device=DEV)
    q = c.q.to(DEV)
    src = new[0].to(DEV)

    def step():
        kernels.update_kv_buffer_kv4(src, dslots, pool)
        return kernels.flash_decoding_kv4(q, pool, SCALE, tbl, lens, 500, b_req_idx=rows, table_kind="block")

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for s in range(4):
        src.copy_(new[s])
        for how in ("eager", "graph"):
            if how == "eager":
                got = step()
            else:
                g.replay()
                got = captured
            torch.cuda.synchronize()
            K4.append(new[s], slots, c.pool)
            for i in range(3):
                c.values[i] = K4.rows_of(c.pool, c.slots[i])
            want, tol, _ = c.want()
            _within(got, want, tol)
            assert torch.equal(pool.cpu(), c.pool)

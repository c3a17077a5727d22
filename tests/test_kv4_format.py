"""The 4-bit cache's format and refusals without a GPU: the oracle agrees with itself and with the error
bound of the definition, and every entry point refuses what it documents before anything is launched."""

import inspect
import math

import pytest
import torch

from llama_lite_npu_b200 import kernels, workloads as W
from oracle import kv4_oracle as K4


def _rows(seed, n, rows, gain=1.0):
    return (W.hash_normal_fp16(seed, (n, rows, 128), 1).float() * gain).half()


def test_every_element_has_a_place_of_its_own():
    for t in range(16):
        seen = {(int(b), int(h)) for b, h in zip(K4.BYTE[t], K4.HIGH[t])}
        assert len(seen) == 128 and {b for b, _ in seen} == set(range(64 * t, 64 * t + 64))


@pytest.mark.parametrize("gain", [1e-6, 1e-3, 1.0, 30.0, 4000.0])
def test_append_and_read_back_within_half_a_step(gain):
    n, rows = 37, 6
    x = _rows(3, n, rows, gain)
    pool = torch.randint(0, 256, (4, rows, K4.BLOCK), dtype=torch.uint8)
    slots = torch.from_numpy(W.hash_permutation(4, 64, 2)[:n].astype("int32"))
    K4.append(x, slots, pool)
    got = K4.rows_of(pool, slots)
    g = x.double().unflatten(-1, (4, 32))
    amax = g.abs().amax(-1, keepdim=True)
    # half a step of the rounded scale (off by 2^-11 relative, or half the smallest fp16), seven steps of rounding
    step = amax / 7
    tol = 0.5 * step * (1 + 2.0 ** -11) + 7 * torch.maximum(step * 2.0 ** -11, torch.tensor(2.0 ** -25, dtype=torch.float64))
    tol = torch.maximum(tol, torch.where(step < 2.0 ** -25, amax, 0.0))      # the scale rounds to zero
    assert bool(((got.unflatten(-1, (4, 32)) - g).abs() <= tol + 1e-30).all())


def test_special_values():
    x = torch.zeros(5, 2, 128, dtype=torch.float16)
    x[1, 0, 3] = float("inf")
    x[2, 1, 40] = float("nan")
    x[3] = 65504.0
    x[4, 0, :32] = torch.tensor(2.0 ** -24)
    pool = torch.zeros(1, 2, K4.BLOCK, dtype=torch.uint8)
    K4.append(x, torch.arange(5, dtype=torch.int32), pool)
    got = K4.rows_of(pool, torch.arange(5, dtype=torch.int32))
    assert bool((got[0] == 0).all())
    assert bool(got[1, 0, :32].isnan().all()) and bool((got[1, 0, 32:] == 0).all()) and bool((got[1, 1] == 0).all())
    assert bool(got[2, 1, 32:64].isnan().all()) and int(got[2].isnan().sum()) == 32
    assert bool((got[3] == 65464.0).all()) and bool(torch.isfinite(got[3].half()).all())
    assert bool((got[4] == 0).all())


def test_surface_matches_the_fp16_operators():
    """Same parameter names and order as the fp16 operators, the two pool views replaced by the pool."""
    names = lambda f: list(inspect.signature(f).parameters)  # noqa: E731
    swap = lambda n: ["KV4_Buffer" if x == "KV_Buffer" else x for x in n]  # noqa: E731
    assert names(kernels.update_kv_buffer_kv4) == swap(names(kernels.update_kv_buffer))
    assert names(kernels.update_kv_buffer_kv4_split) == swap(names(kernels.update_kv_buffer_split))
    assert names(kernels.fused_qk_norm_rope_append_kv4) == swap(names(kernels.fused_qk_norm_rope_append))
    for fn, ref in ((kernels.flash_decoding_kv4, kernels.flash_decoding),
                    (kernels.paged_chunk_flash_attention_kv4, kernels.paged_chunk_flash_attention)):
        want = ["KV4_Buffer" if x == "k_cache" else x for x in names(ref) if x != "v_cache"]
        assert names(fn) == want


def test_operators_refuse_cpu_tensors():
    pool = kernels.empty_kv4_buffer(2, 1, device="cpu")
    assert pool.shape == (2, 2, 1152) and pool.dtype == torch.uint8
    with pytest.raises(ValueError, match="no CPU fallback"):
        kernels.update_kv_buffer_kv4(torch.zeros(1, 2, 128, dtype=torch.float16), torch.zeros(1, dtype=torch.int32), pool)
    with pytest.raises(ValueError, match="no CPU fallback"):
        kernels.gather_kv_buffer_kv4(pool, torch.zeros(1, dtype=torch.int32))


EINVAL, EUNSUPPORTED, EALIGN, EWORKSPACE, ETOOLARGE = 1, 2, 3, 4, 6
A = 0x10000          # an aligned address that is never dereferenced: every call below is refused first


def _append(lib, k=A, v=A, n=4, ks=512, vs=512, slots=A, pool=A, pages=8, stride=2 * 4 * 1152, kvh=4, d=128):
    return lib.b200kv_kv4_append(k, v, n, ks, vs, slots, pool, pages, stride, kvh, d, None, None)


@pytest.mark.parametrize("kw, code", [
    (dict(n=-1), EINVAL), (dict(kvh=0), EINVAL), (dict(d=64), EUNSUPPORTED), (dict(k=None), EINVAL),
    (dict(v=None), EINVAL), (dict(slots=None), EINVAL), (dict(pool=None), EINVAL), (dict(pages=0), EINVAL),
    (dict(stride=2 * 4 * 1152 - 16), EINVAL), (dict(stride=2 * 4 * 1152 + 8), EALIGN), (dict(ks=511), EALIGN),
    (dict(ks=504), EINVAL), (dict(k=A + 8), EALIGN), (dict(pool=A + 8), EALIGN), (dict(pages=1 << 28), ETOOLARGE),
    (dict(n=1 << 31), ETOOLARGE), (dict(n=0, k=None, pool=None), 0)])
def test_append_refusals(built_lib, kw, code):
    assert _append(built_lib, **kw) == code


@pytest.mark.parametrize("kw, code", [
    (dict(q=None), EINVAL), (dict(kv=None), EINVAL), (dict(cos=None), EINVAL), (dict(qh=0), EINVAL),
    (dict(eps=-1.0), EINVAL), (dict(eps=math.nan), EINVAL), (dict(kvs=2 * 512 - 8), EINVAL), (dict(qs=8 * 128 - 8), EINVAL),
    (dict(cs=56), EINVAL), (dict(cs=60), EALIGN), (dict(qw=A + 2), EALIGN), (dict(d=64), EUNSUPPORTED), (dict(n=0), 0)])
def test_fused_append_refusals(built_lib, kw, code):
    a = dict(q=A, qs=8 * 128, kv=A, kvs=2 * 512, qw=A, kw=A, eps=1e-6, cos=A, cs=128, n=4, qh=8, kvh=4, d=128)
    a.update(kw)
    assert built_lib.b200kv_kv4_qk_norm_rope_append(
        a["q"], a["q"], a["qs"], a["qs"], a["kv"], a["kvs"], a["qw"], a["kw"], a["eps"], a["cos"], a["cos"], a["cs"], A,
        A, 8, 2 * 4 * 1152, a["n"], a["qh"], a["kvh"], a["d"], None, None) == code


@pytest.mark.parametrize("kw, code", [
    (dict(n=-1), EINVAL), (dict(out=None), EINVAL), (dict(slots=None), EINVAL), (dict(out=A + 8), EALIGN),
    (dict(os=8 * 128 - 8), EINVAL), (dict(os=8 * 128 + 4), EALIGN), (dict(kvh=0), EINVAL), (dict(n=0), 0)])
def test_gather_refusals(built_lib, kw, code):
    a = dict(n=4, out=A, slots=A, os=8 * 128, kvh=4)
    a.update(kw)
    assert built_lib.b200kv_kv4_gather(A, 8, 2 * 4 * 1152, a["slots"], a["n"], a["out"], a["os"], a["kvh"], 128, None,
                                       None) == code


@pytest.mark.parametrize("kw, code", [
    (dict(batch=0), 0), (dict(batch=-1), EINVAL), (dict(q=None), EINVAL), (dict(table=None), EINVAL),
    (dict(lens=None), EINVAL), (dict(out=None), EINVAL), (dict(ws=None), EINVAL), (dict(kind=2), EINVAL),
    (dict(d=64), EUNSUPPORTED), (dict(ps=32), EUNSUPPORTED), (dict(qh=9), EUNSUPPORTED), (dict(qh=68), EUNSUPPORTED),
    (dict(batch=4097), ETOOLARGE), (dict(cols=0), EINVAL), (dict(rows=1), EINVAL), (dict(max_len=10 * 16 + 1), EINVAL),
    (dict(max_len=-1), EINVAL), (dict(flags=2), EINVAL), (dict(q=A + 8), EALIGN), (dict(qsb=1028), EALIGN),
    (dict(osb=1026), EALIGN), (dict(pages=0), EINVAL)])
def test_decode_refusals(built_lib, kw, code):
    a = dict(q=A, qsb=1024, batch=2, qh=8, kvh=4, d=128, ps=16, table=A, rows=2, cols=10, kind=0, lens=A, max_len=160,
             ws=A, wsb=1 << 30, out=A, osb=1024, flags=0, pages=8)
    a.update(kw)
    assert built_lib.b200kv_kv4_paged_decode(
        a["q"], a["qsb"], 128, A, a["pages"], 2 * 4 * 1152, a["table"], a["cols"], a["kind"], a["rows"], a["cols"], None,
        a["lens"], 0, a["batch"], a["qh"], a["kvh"], a["d"], a["ps"], 0.1, a["max_len"], a["ws"], a["wsb"], a["out"],
        a["osb"], 128, a["flags"], None, None) == code


@pytest.mark.parametrize("kw, code", [
    (dict(batch=0), 0), (dict(total=0), 0), (dict(maxq=0), 0), (dict(batch=-1), EINVAL), (dict(q=None), EINVAL),
    (dict(kind=2), EINVAL), (dict(pool=None), EINVAL), (dict(table=None), EINVAL), (dict(ps=8), EUNSUPPORTED),
    (dict(qh=9), EUNSUPPORTED), (dict(os=1028), EALIGN), (dict(pages=0), EINVAL)])
def test_prefill_refusals(built_lib, kw, code):
    a = dict(q=A, pool=A, pages=8, table=A, kind=0, batch=2, total=8, maxq=4, qh=8, ps=16, os=1024)
    a.update(kw)
    assert built_lib.b200kv_kv4_paged_prefill(
        a["q"], 1024, 128, a["pool"], a["pages"], 2 * 4 * 1152, a["table"], 10, a["kind"], 2, 10, A, A, A, A, 0,
        a["batch"], a["total"], a["maxq"], a["qh"], 4, 128, a["ps"], 0.1, A, a["os"], 128, None, 0, None, None) == code


def test_capture_id_wants_a_place_for_the_answer(built_lib):
    assert built_lib.b200kv_stream_capture_id(None, None) == EINVAL


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf")])
@pytest.mark.parametrize("ws", [None, A])
def test_prefill_refuses_a_scale_that_is_not_positive(built_lib, scale, ws):
    assert built_lib.b200kv_kv4_paged_prefill(
        A, 1024, 128, A, 8, 2 * 4 * 1152, A, 10, 0, 2, 10, A, A, A, A, 0, 2, 8, 4, 8, 4, 128, 16, scale, A, 1024, 128, ws,
        0, None, None) == EINVAL


def test_native_calls_refuse_what_is_no_tensor(built_lib):
    """Objects of any kind in place of the pool, and wrong numbers of arguments, raise."""
    import numpy as np

    from llama_lite_npu_b200 import _kv4_native as native

    pool = kernels.empty_kv4_buffer(2, 1, device="cpu")
    with pytest.raises(ValueError):
        kernels.gather_kv_buffer_kv4(pool, torch.zeros(1, dtype=torch.int32))       # connects the module
    counts = {"append": 4, "prologue": 10, "gather": 3, "decode": 11, "prefill": 11}
    for name, n in counts.items():
        fn = getattr(native, name)
        for wrong in (0, 1, n - 1, n + 1):
            with pytest.raises(TypeError):
                fn(*([pool] * wrong))
        for junk in (None, 3, 2.5, "pool", [1, 2], (1, 2, 3), np.zeros((2, 2, 1152), dtype=np.uint8), object(), torch.Tensor):
            with pytest.raises((TypeError, ValueError, AttributeError)):
                fn(*([junk] * n))
    for bad in (None, {}, {"float16": 1}):
        with pytest.raises((TypeError, KeyError)):
            native.setup(bad)

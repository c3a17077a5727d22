"""Seeded random shapes of the 4-bit cache's attention operators against the 64-bit statement: heads, lengths from
none to some thousands, ragged chunks, both tables, both integer types; tolerances as in test_gpu_kv4.py."""

import os
import random

import pytest
import torch

from llama_lite_npu_b200 import kernels
from test_gpu_kv4 import Case, _within

pytestmark = pytest.mark.gpu
SEEDS = int(os.environ.get("B200KV_SWEEP", "20"))


@pytest.fixture(scope="module", autouse=True)
def _lib_loaded(built_lib):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    yield
    kernels.check_status(0)


def _length(rng, top):
    return rng.choice([rng.randint(0, 3), rng.randint(1, 40), rng.randint(1, 400), rng.randint(1, top)])


@pytest.mark.parametrize("seed", range(SEEDS))
def test_decode(seed):
    rng = random.Random(1000 + seed)
    kvh = rng.choice([1, 1, 2, 3, 8])
    qh = kvh * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16] if kvh < 8 else [1, 2, 3])
    c = Case(seed, [_length(rng, 3000) for _ in range(rng.choice([1, 2, 3, 7, 20]))], qh, kvh)
    want, tol, _ = c.want()
    _within(c.decode(rng.choice(["block", "token"]), rng.choice([torch.int32, torch.int64])), want, tol)


@pytest.mark.parametrize("seed", range(SEEDS))
def test_prefill(seed):
    rng = random.Random(2000 + seed)
    kvh = rng.choice([1, 1, 2, 4])
    qh = kvh * rng.choice([1, 2, 3, 4, 8, 16] if kvh < 4 else [1, 2])
    most = rng.choice([3, 20, 130, 300])
    q_lens = [rng.randint(0, most) for _ in range(rng.choice([1, 2, 4]))] + [rng.randint(1, most)]
    lens = [q + (_length(rng, 2500) if q else 0) for q in q_lens]
    c = Case(seed, lens, qh, kvh, q_lens)
    want, _, tol = c.want()
    _within(c.prefill(rng.choice(["block", "token"]), rng.choice([torch.int32, torch.int64])), want, tol)

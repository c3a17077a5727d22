"""The operators of the 4-bit paged KV cache as they are measured: cases, inputs, and each operator in
its plain form (elementary torch operations in 32 bits) or through the package's own entry points.

The cache holds, per page of 16 tokens and per head, 16 rows of 64 bytes of 4-bit codes followed by
16 rows of four fp16 scales.  A group is 32 neighbouring elements of a head row; with
``d = 32 g + 8 j + n`` the code of (token t, element d) is nibble ``n // 2 + 4 (n & 1)`` of the 32-bit
word at byte ``64 t + 16 (j ^ ((t >> 1) & 3)) + 4 g`` and stands for ``scale[t, g] * (code - 8)``.
"""

from __future__ import annotations

import math

import torch

own = False

D = 128                # head_dim
PS = 16                # tokens of a page
GROUP = 32             # elements that share a scale
BLOCK = PS * D // 2 + PS * (D // GROUP) * 2   # bytes of one page of one head: 1152
EPS = 1e-6
LOG2E = 1.4426950408889634
MOST_SCALE = 9352.0    # 7 times it is the largest multiple of 7 scale steps that fp16 holds


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a small model: four sequences, norm + rotation + append, then the rows read back
        dict(name="prologue_step_4", op="prologue", n=4, q_heads=16, kv_heads=8, norm=True, run=1),
        # a packed prefill of a 64/8-head model, odd length, chunks that start inside a page
        dict(name="prologue_prefill_8205", op="prologue", n=8205, q_heads=64, kv_heads=8, norm=True, run=547),
        # a decode step's plain append on a KV-head shard, no rotation
        dict(name="append_step_33", op="append", n=33, q_heads=8, kv_heads=1, norm=False, run=1),
        # a long packed prefill's plain append into a shuffled pool
        dict(name="append_prefill_65536", op="append", n=65536, q_heads=64, kv_heads=8, norm=False, run=2048),
        # one short request's rows fetched for a dense consumer
        dict(name="gather_201", op="gather", n=201, q_heads=32, kv_heads=4, norm=False, run=201),
        # a batch of long contexts moved out of the cache
        dict(name="gather_40000", op="gather", n=40000, q_heads=64, kv_heads=8, norm=False, run=2500),
        # few short sequences: a chat's first answers, where latency counts
        dict(name="decode_b4_short", op="decode", batch=4, q_heads=16, kv_heads=8, lo=64, hi=512, dist="uniform",
             table="token", chunk=1),
        # the ordinary serving batch of a 64/8-head model, contexts of 1 to 4 k tokens
        dict(name="decode_b32_4k", op="decode", batch=32, q_heads=64, kv_heads=8, lo=1024, hi=4096, dist="uniform",
             table="block", chunk=1),
        # long mixed contexts, three decades of lengths in one batch
        dict(name="decode_b48_16k_mixed", op="decode", batch=48, q_heads=64, kv_heads=8, lo=16, hi=16384, dist="log",
             table="block", chunk=1),
        # a handful of tokens per request on top of a long context (drafted tokens, a prompt's last words)
        dict(name="prefill_b8_7_on_2k", op="prefill", batch=8, q_heads=32, kv_heads=4, lo=300, hi=2100,
             dist="uniform", table="token", chunk=7),
        # packed prompts of up to 2048 tokens, part of each in the prefix cache
        dict(name="prefill_b8_prompts", op="prefill", batch=8, q_heads=64, kv_heads=8, lo=128, hi=1024,
             dist="uniform", table="block", chunk=1024),
        # one chunk of a chunked prefill far into a long prompt
        dict(name="prefill_b2_500_on_16k", op="prefill", batch=2, q_heads=32, kv_heads=4, lo=9000, hi=16000,
             dist="uniform", table="block", chunk=500),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prologue", "append", "gather", "decode", "decode", "prefill"])
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16] if kv_heads < 8 else [1, 2, 3, 5, 8])
    if op in ("prologue", "append", "gather"):
        n = _log_int(rng, 1, 16000 if op == "prologue" else 40000)
        return dict(op=op, n=n, q_heads=q_heads, kv_heads=kv_heads, norm=op == "prologue" and rng.random() < 0.6,
                    run=min(n, _log_int(rng, 1, 2500)))
    table = rng.choice(["token", "block"])
    if op == "decode":
        lo = _log_int(rng, 1, 1500)
        return dict(op=op, batch=_log_int(rng, 1, 40), q_heads=q_heads, kv_heads=kv_heads, lo=lo,
                    hi=min(lo * rng.choice([1, 3, 9, 60]), 14000), dist=rng.choice(["uniform", "log"]), table=table,
                    chunk=1)
    lo = _log_int(rng, 1, 3000)
    return dict(op=op, batch=rng.randint(1, 6), q_heads=min(q_heads, 64), kv_heads=kv_heads, lo=lo, hi=2 * lo,
                dist="uniform", table=table, chunk=_log_int(rng, 1, 700))


# ---------------------------------------------------------------------------------------------
# the format in plain operations
# ---------------------------------------------------------------------------------------------
def _quantise(x):
    """fp16 ``[..., 128]`` -> codes 0..15 (uint8 ``[..., 128]``) and scales (fp16 ``[..., 4]``)."""
    g = x.float().unflatten(-1, (D // GROUP, GROUP))
    amax = g.abs().amax(-1)
    scale = (amax / 7.0).half().clamp(max=MOST_SCALE)
    s = scale.double().unsqueeze(-1)                      # 64 bits: values next to a border
    c = torch.floor(torch.where(s > 0, g.double() / s, 0.0) + 0.5).clamp(-8, 7)
    fine = torch.isfinite(amax)
    codes = torch.where(fine.unsqueeze(-1), c + 8, 8.0).to(torch.uint8).flatten(-2)
    return codes, torch.where(fine, scale, float("nan")).half()


def _byte_order(t):
    """For token-in-page numbers ``t`` [n]: which chunk j sits at chunk position p, [n, 4]."""
    return torch.arange(4, device=t.device) ^ ((t.unsqueeze(-1) >> 1) & 3)


def _pack_rows(codes, t):
    """Codes ``[n, rows, 128]`` of tokens at page positions ``t`` [n] -> bytes ``[n, rows, 64]``."""
    n, rows = codes.shape[:2]
    c = codes.view(n, rows, 4, 4, 8).transpose(2, 3)       # [n, rows, j, g, 8]
    c = c.unflatten(-1, (4, 2)).transpose(-1, -2).flatten(-2)   # even elements, then odd ones
    c = c[..., 0::2] | (c[..., 1::2] << 4)                 # [n, rows, j, g, 4 bytes]
    at = _byte_order(t).view(n, 1, 4, 1, 1).expand(n, rows, 4, 4, 4)
    return torch.gather(c, 2, at).reshape(n, rows, 64)


def _nibbles(b):
    """Bytes ``[..., 4]`` of words -> their eight codes in the order of the elements."""
    return torch.stack((b & 15, b >> 4), -1).unflatten(-2, (2, 2)).flatten(-2).transpose(-1, -2).flatten(-2)


def _unpack_blocks(blocks):
    """Blocks ``[..., 1152]`` uint8 -> the values they stand for, fp32 ``[..., 16, 128]``."""
    b = blocks[..., : PS * 64].unflatten(-1, (PS, 4, 4, 4))
    t = torch.arange(PS, device=blocks.device)
    b = b[..., t.unsqueeze(-1), _byte_order(t), :, :]      # [..., 16, j, g, 4 bytes]
    c = _nibbles(b).transpose(-3, -2).flatten(-2).float() - 8   # [..., 16, g, 32]
    s = blocks[..., PS * 64:].contiguous().view(torch.float16).unflatten(-1, (PS, 4)).float()
    return (c * s.unsqueeze(-1)).flatten(-2)


def _plain_append(rows, slots, pool):
    """Quantises fp16 ``rows`` [n, 2*kv_heads, 128] into the pool's slots."""
    codes, scales = _quantise(rows)
    page, t = slots.long() // PS, slots.long() % PS
    pool[..., : PS * 64].unflatten(-1, (PS, 64))[page, :, t] = _pack_rows(codes, t)
    pool.view(torch.float16)[..., PS * 32:].unflatten(-1, (PS, 4))[page, :, t] = scales


def _plain_gather(pool, slots):
    page, t = slots.long() // PS, slots.long() % PS
    rows = pool[..., : PS * 64].unflatten(-1, (PS, 4, 4, 4))[page, :, t]            # [n, rows, 4, 4, 4]
    n, r = rows.shape[:2]
    rows = torch.gather(rows, 2, _byte_order(t).view(n, 1, 4, 1, 1).expand_as(rows))
    c = _nibbles(rows).transpose(2, 3).reshape(n, r, 4, 32).float() - 8
    s = pool.view(torch.float16)[..., PS * 32:].unflatten(-1, (PS, 4))[page, :, t].float()
    return (c * s.unsqueeze(-1)).flatten(-2).half()


def _plain_norm(x, weight):
    """RMSNorm of fp16 head rows: statistics in 64 bits, x * rrms and the weighted value each rounded to fp16."""
    ms = (x.double().square().sum(-1, keepdim=True) / D).float()
    return (x.float() * (1.0 / torch.sqrt(ms + EPS))).half() * weight


def _plain_rotate(x, cos, sin):
    a, b = x[..., : D // 2].float(), x[..., D // 2:].float()
    c, s = cos[:, None, : D // 2].float(), sin[:, None, : D // 2].float()
    return torch.cat((a * c - b * s, b * c + a * s), -1).half()


def _padded_kv(st):
    """K and V of every sequence, padded to the longest: fp32 [batch, kv_heads, positions, 128] each."""
    pages = st["block_table"][st["rows"].long()].long()
    x = _unpack_blocks(st["pool"][pages])                              # [b, pages, 2*kvh, 16, 128]
    x = x.permute(2, 0, 1, 3, 4).flatten(2, 3)                         # [2*kvh, b, positions, 128]
    here = torch.arange(x.shape[2], device=x.device) < st["kv_lens"].unsqueeze(-1)
    x = torch.where(here.unsqueeze(-1), x, 0.0)
    kvh = x.shape[0] // 2
    return x[:kvh].transpose(0, 1), x[kvh:].transpose(0, 1)


def _plain_attention(st):
    """Attention of every query row over its request's keys up to its own position."""
    k, v = _padded_kv(st)
    b, kvh, positions, _ = k.shape
    q, b_of, i_of = st["q"], st["row_request"], st["row_index"]
    group = q.shape[1] // kvh
    padded = torch.zeros(b, st["chunk"], q.shape[1], D, device=q.device)
    padded[b_of, i_of] = q.float()
    x = padded.unflatten(2, (kvh, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)     # [b, kvh, group*chunk, 128]
    s = (x @ k.transpose(-1, -2)).unflatten(2, (group, st["chunk"])) * (1.0 / math.sqrt(D))
    last = (st["kv_lens"] - st["q_lens"]).unsqueeze(-1) + torch.arange(st["chunk"], device=q.device)
    seen = torch.arange(positions, device=q.device) <= last.unsqueeze(-1)            # [b, chunk, positions]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    s = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    o = s.flatten(2, 3) @ v / s.sum(-1).flatten(2, 3).unsqueeze(-1)
    o = o.unflatten(2, (group, st["chunk"])).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [b, chunk, heads, 128]
    return o[b_of, i_of].half()


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _kv_rows(n, kv_heads, gen):
    """K and V rows as projections give them: some channels of K are much larger than the others."""
    x = torch.randn(n, 2 * kv_heads, D, device="cuda", generator=gen)
    gain = torch.exp(0.5 * torch.randn(2 * kv_heads, D, device="cuda", generator=gen))
    gain[kv_heads:] = 0.5
    return x.mul_(gain).half()


def _lengths(case, gen):
    # one length from each of `batch` equal parts of the distribution, in any order
    part = torch.randperm(case["batch"], generator=gen, device="cuda").double()
    u = ((part + torch.rand(case["batch"], generator=gen, device="cuda", dtype=torch.float64)) / case["batch"]).cpu()
    lo, hi = case["lo"], max(case["lo"], case["hi"])
    if case["dist"] == "log":
        n = torch.exp(math.log(lo) + u * (math.log(hi + 1) - math.log(lo))).floor().long()
    else:
        n = (lo + u * (hi + 1 - lo)).floor().long()
    return n.clamp(lo, hi)


def _query_lengths(case):
    """Query rows of each request: a chunk's requests bring between half of it and all of it."""
    chunk = case["chunk"]
    return [max(1, chunk - int(i * 0.618034 % 1.0 * chunk / 2)) for i in range(case["batch"])]


def _random_pool(pages, kv_heads, gen):
    return torch.randint(0, 256, (pages, 2 * kv_heads, BLOCK), dtype=torch.uint8, device="cuda", generator=gen)


def _row_case(case, gen):
    """Inputs of the append and gather operators: n rows in runs of neighbouring tokens, the runs on
    shuffled pages and starting anywhere in a page."""
    n, kvh, qh, run = case["n"], case["kv_heads"], case["q_heads"], case["run"]
    runs = -(-n // run)
    per_run = (run + 2 * PS - 2) // PS
    pages = runs * per_run + 3
    order = torch.randperm(pages, device="cuda", generator=gen)
    first = torch.randint(0, PS, (runs, 1), device="cuda", generator=gen)
    pos = first + torch.arange(run, device="cuda")
    which = torch.arange(runs, device="cuda").unsqueeze(-1) * per_run + pos // PS
    slots = (order[which] * PS + pos % PS).reshape(-1)[:n].int().contiguous()
    st = dict(op=case["op"], slots=slots, pool=_random_pool(pages, kvh, gen))
    rows = _kv_rows(n, kvh, gen)
    if case["op"] == "gather":
        _plain_append(rows, slots, st["pool"])
        return st
    st["kv"] = rows
    if case["op"] == "prologue":
        st["q"] = torch.randn(n, qh, D, device="cuda", generator=gen).half()
        place = torch.randint(0, 30000, (n, 1), device="cuda", generator=gen).double()
        angle = place * 1e6 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))
        st["cos"], st["sin"] = (torch.cat((f(angle),) * 2, -1).half() for f in (torch.cos, torch.sin))
        for w in ("q_weight", "k_weight"):
            st[w] = (1 + 0.2 * torch.randn(D, device="cuda", generator=gen)).half() if case["norm"] else None
    return st


def _attention_case(case, gen):
    """A pool on shuffled pages with the sequences' tables.  What lies behind a sequence's last token
    in its last page was never written: random bytes."""
    b, kvh, qh = case["batch"], case["kv_heads"], case["q_heads"]
    lens = _lengths(case, gen)
    q_lens = torch.ones(b, dtype=torch.long)
    if case["op"] == "prefill":      # lengths are the contexts; the chunks differ from request to request
        q_lens = torch.tensor(_query_lengths(case))
        lens = lens + q_lens
    pages = (lens + PS - 1) // PS
    width, total = int(pages.max()), int(pages.sum())
    order = torch.randperm(total + 2, device="cuda", generator=gen)
    at = torch.arange(width).unsqueeze(0)
    index = ((pages.cumsum(0) - pages).unsqueeze(-1) + at).clamp(max=total - 1).cuda()
    listed_page = (at < pages.unsqueeze(-1)).cuda()
    by_batch = torch.where(listed_page, order[index], 0)
    rows = torch.randperm(b + 2, device="cuda", generator=gen)[:b]     # table rows in another order, with gaps
    block_table = torch.zeros(b + 2, width, dtype=torch.int32, device="cuda")
    block_table[rows] = by_batch.int()
    token_table = (block_table.unsqueeze(-1) * PS + torch.arange(PS, device="cuda", dtype=torch.int32)).flatten(1)
    pool = _random_pool(total + 2, kvh, gen)
    lens_dev = lens.cuda()
    pos = torch.arange(width * PS, device="cuda")
    live = pos < lens_dev.unsqueeze(-1)
    slots = token_table[rows][live]
    part = 1 << 17
    for i in range(0, slots.shape[0], part):
        _plain_append(_kv_rows(min(part, slots.shape[0] - i), kvh, gen), slots[i: i + part], pool)
    n_q = int(q_lens.sum())
    start = q_lens.cumsum(0) - q_lens
    request = torch.repeat_interleave(torch.arange(b), q_lens)
    return dict(op=case["op"], pool=pool, block_table=block_table, token_table=token_table.contiguous(),
                table=case["table"], rows=rows.int(), kv_lens=lens_dev, q_lens=q_lens.cuda(),
                ctx_lens=(lens - q_lens).cuda(), q_start=start.int().cuda(), chunk=int(q_lens.max()),
                max_len=int(lens.max()), row_request=request.cuda(),
                row_index=(torch.arange(n_q) - start[request]).cuda(),
                q=(1.5 * torch.randn(n_q, qh, D, device="cuda", generator=gen)).half())


def prepare(case, seed):
    gen = _generator(seed)
    return _row_case(case, gen) if case["op"] in ("prologue", "append", "gather") else _attention_case(case, gen)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(st):
    op = st["op"]
    if own:
        from llama_lite_npu_b200 import kernels

        if op == "gather":
            return kernels.gather_kv_buffer_kv4(st["pool"], st["slots"])
        if op == "append":
            kernels.update_kv_buffer_kv4(st["kv"], st["slots"], st["pool"])
            return kernels.gather_kv_buffer_kv4(st["pool"], st["slots"])
        if op == "prologue":
            q = kernels.fused_qk_norm_rope_append_kv4(
                st["q"], st["kv"].flatten(1), st["q_weight"], st["k_weight"], EPS, st["cos"], st["sin"], st["slots"],
                st["pool"], out=torch.empty_like(st["q"]))
            return q, kernels.gather_kv_buffer_kv4(st["pool"], st["slots"])
        table = st["token_table"] if st["table"] == "token" else st["block_table"]
        if op == "decode":
            return kernels.flash_decoding_kv4(
                st["q"], st["pool"], 1.0 / math.sqrt(D), table, st["kv_lens"], st["max_len"], b_req_idx=st["rows"],
                table_kind=st["table"])
        return kernels.paged_chunk_flash_attention_kv4(
            st["q"], st["pool"], LOG2E / math.sqrt(D), table, st["rows"], st["q_start"], st["ctx_lens"], st["q_lens"],
            st["chunk"], table_kind=st["table"])
    if op == "gather":
        return _plain_gather(st["pool"], st["slots"])
    if op == "append":
        _plain_append(st["kv"], st["slots"], st["pool"])
        return _plain_gather(st["pool"], st["slots"])
    if op == "prologue":
        kvh = st["kv"].shape[1] // 2
        q, k, v = st["q"], st["kv"][:, :kvh], st["kv"][:, kvh:]
        if st["q_weight"] is not None:
            q, k = _plain_norm(q, st["q_weight"]), _plain_norm(k, st["k_weight"])
        q, k = (_plain_rotate(x, st["cos"], st["sin"]) for x in (q, k))
        _plain_append(torch.cat((k, v), 1), st["slots"], st["pool"])
        return q, _plain_gather(st["pool"], st["slots"])
    return _plain_attention(st)


def work(case):
    row16, row4 = 2 * case["kv_heads"] * D * 2, 2 * case["kv_heads"] * (D // 2 + D // GROUP * 2)
    if case["op"] in ("prologue", "append", "gather"):
        n = case["n"]
        bytes_ = n * (row4 + row16 + 4)                              # the rows read back
        if case["op"] != "gather":
            bytes_ += n * (row16 + row4 + 4)
        if case["op"] == "prologue":
            bytes_ += n * (2 * case["q_heads"] * D * 2 + 2 * D)      # Q in and out, half a row of cos and of sin
        return {"bytes": float(bytes_), "flops": float(4 * n * (case["kv_heads"] + case["q_heads"]) * D)}
    # the mean of the lengths that are drawn
    lo, hi = case["lo"], max(case["lo"], case["hi"])
    mean = (hi - lo) / math.log(hi / lo) if case["dist"] == "log" and hi > lo else (lo + hi) / 2
    ctx = mean - 1 if case["op"] == "decode" else mean
    bytes_ = flops = 0.0
    for q in _query_lengths(case):
        kv = ctx + q
        bytes_ += kv * row4 + kv / PS * 4 + 2 * q * case["q_heads"] * D * 2
        flops += 4.0 * D * case["q_heads"] * (q * ctx + q * (q + 1) / 2)
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_values(pool, slots):
    """Values of pool rows by the address of every code: fp64 [n, rows, 128]."""
    d = torch.arange(D, device=pool.device)
    g, j, n = d // 32, d % 32 // 8, d % 8
    page, t = slots.long().unsqueeze(-1) // PS, slots.long().unsqueeze(-1) % PS
    nibble = n // 2 + 4 * (n % 2)
    byte = 64 * t + 16 * (j ^ (t // 2 % 4)) + 4 * g + nibble // 2               # [n, 128]
    scale_at = PS * 64 + 8 * t + 2 * g
    flat = pool.view(-1)
    rows = torch.arange(pool.shape[1], device=pool.device).view(1, -1, 1)
    base = (page.unsqueeze(-1) * pool.shape[1] + rows) * BLOCK
    code = (flat[base + byte.unsqueeze(1)].long() >> (4 * (nibble % 2))) & 15
    scale = pool.view(torch.float16).view(-1)[(base + scale_at.unsqueeze(1)) // 2]
    return (code - 8).double() * scale.double()


def _exact_stored(x):
    """What the cache stands for after fp16 values ``x`` were appended: fp64, same shape."""
    g = x.double().view(*x.shape[:-1], D // GROUP, GROUP)
    scale = (g.abs().max(-1).values / 7).half().double().clamp(max=MOST_SCALE).unsqueeze(-1)
    c = torch.where(scale == 0, torch.zeros_like(g), torch.floor(g / scale + 0.5)).clamp(-8, 7)
    return (c * scale).view(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    op = st["op"]
    if op == "gather":
        return _exact_values(st["pool"], st["slots"])
    if op == "append":
        return _exact_stored(st["kv"])
    if op == "prologue":
        kvh = st["kv"].shape[1] // 2
        x = torch.cat((st["q"], st["kv"][:, :kvh]), 1).double()
        if case["norm"]:      # the two roundings to fp16 inside the norm are part of its definition
            x = (x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()).half().double()
            qh = st["q"].shape[1]
            x = torch.cat((x[:, :qh] * st["q_weight"].double(), x[:, qh:] * st["k_weight"].double()), 1).half().double()
        turned = torch.complex(x[..., : D // 2], x[..., D // 2:]) * torch.complex(
            st["cos"][:, None, : D // 2].double(), st["sin"][:, None, : D // 2].double())
        x = torch.cat((turned.real, turned.imag), -1)
        q, k = x[:, : st["q"].shape[1]], x[:, st["q"].shape[1]:].half()
        return q, _exact_stored(torch.cat((k, st["kv"][:, kvh:]), 1))
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    kvh = st["pool"].shape[1] // 2
    group = st["q"].shape[1] // kvh
    begin = 0
    for b in range(case["batch"]):
        n, n_q = int(st["kv_lens"][b]), int(st["q_lens"][b])
        x = _exact_values(st["pool"], st["token_table"][int(st["rows"][b]), :n])
        q = st["q"][begin: begin + n_q].double()
        later = torch.arange(n, device="cuda") > (n - n_q) + torch.arange(n_q, device="cuda").unsqueeze(-1)
        for h in range(kvh):
            s = torch.einsum("igd,nd->gin", q[:, h * group: (h + 1) * group], x[:, h]) / math.sqrt(D)
            s[:, later] = -math.inf
            out[begin: begin + n_q, h * group: (h + 1) * group] = (torch.softmax(s, -1) @ x[:, kvh + h]).transpose(0, 1)
        begin += n_q
    return out

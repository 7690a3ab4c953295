# SPDX-License-Identifier: Apache-2.0
"""Measured cases of the operators behind parallel sampling with scored answers.

One prompt is continued by many requests at once, and every token comes with
its log-probability. Four operators run per step:

``layout``    block tables, slot maps and token positions from request lengths
``prefix``    decode attention of a batch whose groups share their prompt's pages
``logprobs``  log-probabilities, ranks, entropy and top alternatives from logits
``score``     the same for given tokens from hidden states, without the logits

With ``own`` false, :func:`run` computes each in elementary torch operations in
32 bits; with ``own`` true it calls the library through its Python binding.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BF16, MX = 0, 1             # page formats: bf16, E4M3 payload with one E4M3 scale per 8 elements
MAX_TOP = 32


# ---------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------

def listed():
    return [
        # a few samples of one short chat prompt, first tokens of the answers: latency
        dict(name="prefix_b8_p512", op="prefix", seqs=8, prefix=512, suffix=64, groups=1,
             hq=32, hkv=8, d=128, kv=MX, block=16),
        # best-of-64 over one long document, answers of up to a thousand tokens
        dict(name="prefix_b64_p8192", op="prefix", seqs=64, prefix=8192, suffix=1024, groups=1,
             hq=32, hkv=8, d=128, kv=MX, block=16),
        # five prompts with ragged sample counts, bf16 pages, group of three query heads
        dict(name="prefix_b77_g5_bf16", op="prefix", seqs=77, prefix=3001, suffix=200, groups=5,
             hq=24, hkv=8, d=128, kv=BF16, block=32),
        # a full continuous batch under one system prompt
        dict(name="prefix_b256_p8192", op="prefix", seqs=256, prefix=8192, suffix=256, groups=1,
             hq=32, hkv=8, d=128, kv=MX, block=16),
        # one decode step of a small batch: every row adds a token
        dict(name="layout_b16_step", op="layout", seqs=16, blocks=128, block=16, new=1, fork=0),
        # a scheduler step with chunked prompts, forks and decode rows mixed
        dict(name="layout_b4096_mixed", op="layout", seqs=4096, blocks=1024, block=16, new=257,
             fork=4),
        # the log-probability of one sampled token with 20 alternatives: latency
        dict(name="logprobs_r1_v128256", op="logprobs", rows=1, vocab=128256, dtype="f32",
             stride=128256, targets=1, top=20, masked=0),
        # a decode batch's logits, as the lm_head writes them
        dict(name="logprobs_r256_v128256", op="logprobs", rows=256, vocab=128256, dtype="f32",
             stride=128256, targets=1, top=20, masked=5),
        # bf16 logits with an odd vocabulary, padded rows and several targets a row
        dict(name="logprobs_r999_v32003_bf16", op="logprobs", rows=999, vocab=32003,
             dtype="bf16", stride=32016, targets=3, top=5, masked=7),
        # a short candidate answer: the vocabulary matrix is read once for 24 rows
        dict(name="score_r24_h4096_v128256", op="score", rows=24, hidden=4096, vocab=128256,
             targets=1, top=20),
        # an odd chunk against a small vocabulary
        dict(name="score_r333_h1024_v32003", op="score", rows=333, hidden=1024, vocab=32003,
             targets=1, top=5),
        # a 2,048-token prompt scored in one call
        dict(name="score_r2048_h4096_v128256", op="score", rows=2048, hidden=4096, vocab=128256,
             targets=1, top=20),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prefix", "prefix", "layout", "logprobs", "logprobs", "score"])
    if op == "prefix":
        hq, hkv, d = rng.choice([(32, 8, 128), (24, 8, 128), (64, 8, 128), (16, 2, 64), (8, 8, 64),
                                 (12, 12, 128)])
        seqs = _log_int(rng, 2, 256)
        suffix = _log_int(rng, 1, 1024)
        # no more than the largest listed case's rows x context, heads and dims counted
        most = 256 * 8320 * 32 * 128 // (hq * d * seqs) - suffix
        prefix = _log_int(rng, 16, max(17, min(16384, most)))
        return dict(op=op, seqs=seqs, prefix=prefix, suffix=suffix,
                    groups=rng.randint(1, min(6, seqs)), hq=hq, hkv=hkv, d=d,
                    kv=rng.choice([MX, MX, BF16]), block=rng.choice([16, 32, 64, 128]))
    if op == "layout":
        block = rng.choice([5, 16, 32, 128])
        return dict(op=op, seqs=_log_int(rng, 1, 4096), blocks=_log_int(rng, 16, 1024),
                    block=block, new=_log_int(rng, 1, 257), fork=rng.choice([0, 3, 8]))
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 160000)
        return dict(op=op, rows=_log_int(rng, 1, 256), vocab=vocab,
                    dtype=rng.choice(["f32", "bf16"]), stride=vocab + rng.choice([0, 1, 13]),
                    targets=rng.randint(1, 4), top=rng.randint(0, MAX_TOP),
                    masked=rng.choice([0, 3]))
    hidden = 64 * _log_int(rng, 4, 64)
    vocab = _log_int(rng, 1000, 128256)
    rows = _log_int(rng, 1, 2048)
    return dict(op=op, rows=rows, hidden=hidden, vocab=vocab, targets=rng.randint(1, 3),
                top=rng.randint(0, MAX_TOP))


# ---------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _page_bytes(c):
    return c["hkv"] * c["block"] * (c["d"] * 9 // 8 if c["kv"] == MX else c["d"] * 2)


def _prefix_shape(c, seed):
    """Row counts of the groups, prefix tokens of each, context length of each row."""
    rs = np.random.RandomState((int(seed) * 31 + 5) % (1 << 31))
    S, G = c["seqs"], c["groups"]
    cuts = np.sort(rs.choice(np.arange(1, S), G - 1, replace=False)) if G > 1 else np.zeros(0, int)
    starts = np.concatenate([[0], cuts, [S]]).astype(np.int64)
    plens = np.full(G, c["prefix"], np.int64)
    for g in range(1, G):
        plens[g] = max(1, c["prefix"] * rs.randint(1, 5) // 4)
    lens = np.zeros(S, np.int64)
    for g in range(G):
        n = starts[g + 1] - starts[g]
        lens[starts[g]:starts[g + 1]] = plens[g] + rs.randint(1, c["suffix"] + 1, n)
    if S >= 16:
        lens[S // 2] = 0                 # a row whose request has ended
    return starts, plens, lens


def _mx_pages(n_pages, c, gen):
    """n_pages MX pages of normal values with per-head magnitudes."""
    H, bs, d = c["hkv"], c["block"], c["d"]
    mag = 0.5 + 3.5 * torch.rand((1, H, 1, 1, 1), generator=gen, device="cuda")
    x = torch.randn((n_pages, H, bs, d // 8, 8), generator=gen, device="cuda") * mag
    scale = (x.abs().amax(-1, keepdim=True) / 448.0).clamp_min(2.0 ** -9).to(torch.float8_e4m3fn)
    pay = (x / scale.float()).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return torch.cat([pay.view(torch.uint8).reshape(n_pages, H, bs * d),
                      scale.view(torch.uint8).reshape(n_pages, H, bs * d // 8)], 2).reshape(n_pages, -1)


def _bf16_pages(n_pages, c, gen):
    H, bs, d = c["hkv"], c["block"], c["d"]
    mag = 0.5 + 3.5 * torch.rand((1, H, 1, 1), generator=gen, device="cuda")
    x = (torch.randn((n_pages, H, bs, d), generator=gen, device="cuda") * mag).bfloat16()
    return x.view(torch.uint8).reshape(n_pages, -1)


def _prepare_prefix(c, seed):
    gen = _gen(seed)
    starts, plens, lens = _prefix_shape(c, seed)
    bs, S = c["block"], c["seqs"]
    nblk = -(-lens // bs)
    max_blocks = int(max(1, nblk.max()))
    shared = plens // bs                                  # whole shared pages of each group
    group = np.repeat(np.arange(len(plens)), np.diff(starts))
    page = np.full((S, max_blocks), -1, np.int64)
    used = 0
    for g in range(len(plens)):
        ids = np.arange(used, used + shared[g])
        used += shared[g]
        for s in range(starts[g], starts[g + 1]):
            k = min(shared[g], nblk[s])
            page[s, :k] = ids[:k]
    for s in range(S):
        own_blocks = max(0, nblk[s] - shared[group[s]])
        page[s, nblk[s] - own_blocks:nblk[s]] = np.arange(used, used + own_blocks)
        used += own_blocks
    n_slots = max(1, used)
    pb = _page_bytes(c)
    make = _mx_pages if c["kv"] == MX else _bf16_pages
    arena = torch.empty((n_slots, 2, pb), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 28) // (pb * 2))
    for a in range(0, n_slots, step):
        b = min(n_slots, a + step)
        for which in range(2):
            arena[a:b, which] = make(b - a, c, gen)
    perm = torch.randperm(n_slots, generator=gen, device="cuda")
    page_t = torch.from_numpy(page).cuda()
    valid = page_t >= 0
    slot = perm[page_t.clamp_min(0)]
    base = arena.data_ptr()
    table = torch.stack([(base + slot * 2 * pb) * valid, (base + slot * 2 * pb + pb) * valid,
                         valid.long()], -1).contiguous()
    q = torch.randn((S, c["hq"], c["d"]), generator=gen, device="cuda").bfloat16()
    return dict(case=c, arena=arena, table=table, q=q, max_blocks=max_blocks,
                lens=torch.from_numpy(lens.astype(np.int32)).cuda(),
                starts=torch.from_numpy(starts.astype(np.int32)).cuda(),
                plens=torch.from_numpy(plens.astype(np.int32)).cuda(),
                out=torch.zeros((S, c["hq"], c["d"]), dtype=torch.bfloat16, device="cuda"),
                err=torch.zeros(1, dtype=torch.int32, device="cuda"))


#: The arena of the layout cases: the entries are addresses that nothing there reads.
_BASE, _SLOT_BYTES, _K_OFF, _V_OFF = 1 << 40, 36864, 0, 18432


def _layout_shape(c, seed):
    rs = np.random.RandomState((int(seed) * 131 + 7) % (1 << 31))
    n, cap = c["seqs"], c["blocks"] * c["block"]
    ctx = np.exp(rs.uniform(0, math.log(max(2, cap - c["new"])), n)).astype(np.int64)
    new = np.ones(n, np.int64) if c["new"] == 1 else np.where(
        rs.rand(n) < 0.5, 1, rs.randint(0, c["new"] + 1, n))
    new = np.minimum(new, cap - ctx)
    fork = np.full(n, -1, np.int64)
    if c["fork"]:
        for s in range(1, n):
            if rs.randint(0, c["fork"]) == 0:
                p = rs.randint(0, s)
                if fork[p] < 0:
                    fork[s] = p
                    ctx[s] = ctx[p] // c["block"] * c["block"]
                    new[s] = min(max(new[s], 1), cap - ctx[s])
    return ctx, new, fork


def _layout_capacity(c):
    """Token rows of a step: later launches of a fixed size take them padded."""
    return 8 + c["seqs"] * (c["new"] + 1) // 2


def _prepare_layout(c, seed):
    ctx, new, fork = _layout_shape(c, seed)
    n, mb, bs = c["seqs"], c["blocks"], c["block"]
    gen = _gen(seed)
    old = -(-ctx // bs)
    held = np.where(fork >= 0, 0, old)
    need = -(-(ctx + new) // bs) - old
    total = int(held.sum() + need.sum() + 64)
    perm = torch.randperm(total, generator=gen, device="cuda")
    first = torch.from_numpy(np.cumsum(held) - held).cuda()
    j = torch.arange(mb, device="cuda")
    has = j[None, :] < torch.from_numpy(held).cuda()[:, None]
    slot = perm[(first[:, None] + j[None, :]).clamp_max(total - 1)]
    addr = _BASE + slot * _SLOT_BYTES
    table = torch.stack([(addr + _K_OFF) * has, (addr + _V_OFF) * has, has.long()], -1).contiguous()
    cap = _layout_capacity(c)
    i32 = dict(dtype=torch.int32, device="cuda")
    up = lambda a: torch.from_numpy(a.astype(np.int32)).cuda()  # noqa: E731
    return dict(case=c, ctx=up(ctx), new=up(new), fork=up(fork), total=total, cap=cap,
                free=perm[int(held.sum()):].to(torch.int32).contiguous(), table=table,
                seq_lens=torch.zeros(n, **i32), cu=torch.zeros(n + 1, **i32),
                token_seq=torch.zeros(cap, **i32), token_pos=torch.zeros(cap, **i32),
                slot_map=torch.zeros(cap, dtype=torch.int64, device="cuda"),
                counts=torch.zeros(2, **i32), err=torch.zeros(1, **i32))


def _prepare_logprobs(c, seed):
    gen = _gen(seed)
    R, V, nt, top = c["rows"], c["vocab"], c["targets"], c["top"]
    dt = torch.float32 if c["dtype"] == "f32" else torch.bfloat16
    buf = torch.full((R, c["stride"]), float("nan"), dtype=dt, device="cuda")
    step = max(1, (1 << 27) // V)
    for a in range(0, R, step):
        b = min(R, a + step)
        x = torch.randn((b - a, V), generator=gen, device="cuda") * 2.5
        peak = torch.randint(0, V, (b - a, 4), generator=gen, device="cuda")
        x.scatter_add_(1, peak, 4 + 8 * torch.rand((b - a, 4), generator=gen, device="cuda"))
        if c["masked"]:                                  # rows under a grammar: few tokens allowed
            keep = torch.rand((b - a, V), generator=gen, device="cuda") < 200.0 / V
            rows = torch.arange(a, b, device="cuda")[:, None]
            x = torch.where((rows % c["masked"] == 1) & ~keep, float("-inf"), x)
        buf[a:b, :V] = x.to(dt)
    tgt = torch.randint(0, V, (R, nt), generator=gen, device="cuda", dtype=torch.int32)
    temp = (0.5 + torch.rand(R, generator=gen, device="cuda")).round(decimals=2)
    return dict(case=c, logits=buf, targets=tgt, temperature=temp, **_score_outputs(R, nt, top))


def _score_outputs(R, nt, top):
    f32 = dict(dtype=torch.float32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(o_lp=torch.zeros((R, nt), **f32), o_rank=torch.zeros((R, nt), **i32),
                o_ent=torch.zeros(R, **f32), o_lse=torch.zeros(R, **f32),
                o_ids=torch.zeros((R, max(1, top)), **i32),
                o_top=torch.zeros((R, max(1, top)), **f32),
                err=torch.zeros(1, **i32))


def _prepare_score(c, seed):
    # Values on a grid of powers of two, so that every sum of products is exact
    # in 32 bits whatever its order: equal and near-equal logits keep their order.
    gen = _gen(seed)
    R, K, V = c["rows"], c["hidden"], c["vocab"]
    h = (torch.randn((R, K), generator=gen, device="cuda") * 8).round().clamp(-32, 32) / 4
    w = torch.empty((V, K), dtype=torch.bfloat16, device="cuda")
    unit = 10.0 * math.sqrt(4096.0 / K)
    step = max(1, (1 << 27) // K)
    for a in range(0, V, step):
        b = min(V, a + step)
        w[a:b] = ((torch.randn((b - a, K), generator=gen, device="cuda") * unit).round()
                  .clamp(-127, 127) / 512).bfloat16()
    tgt = torch.randint(0, V, (R, c["targets"]), generator=gen, device="cuda", dtype=torch.int32)
    temp = (0.5 + torch.rand(R, generator=gen, device="cuda")).round(decimals=2)
    return dict(case=c, hidden=h.bfloat16(), weight=w, targets=tgt, temperature=temp,
                **_score_outputs(R, c["targets"], c["top"]))


def prepare(case, seed):
    return {"prefix": _prepare_prefix, "layout": _prepare_layout,
            "logprobs": _prepare_logprobs, "score": _prepare_score}[case["op"]](dict(case), seed)


# ---------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------

def _pages_f32(pages, c):
    """uint8 [..., page bytes] -> fp32 [..., hkv, block, d]."""
    H, bs, d = c["hkv"], c["block"], c["d"]
    lead = pages.shape[:-1]
    if c["kv"] == BF16:
        return pages.contiguous().view(torch.bfloat16).reshape(*lead, H, bs, d).float()
    sec = pages.reshape(*lead, H, bs * d * 9 // 8)
    pay = sec[..., :bs * d].contiguous().view(torch.float8_e4m3fn).reshape(*lead, H, bs, d // 8, 8)
    sc = sec[..., bs * d:].contiguous().view(torch.float8_e4m3fn).reshape(*lead, H, bs, d // 8, 1)
    return (pay.float() * sc.float()).reshape(*lead, H, bs, d)


def _plain_prefix(st):
    c = st["case"]
    S, H, d, bs, mb = c["seqs"], c["hkv"], c["d"], c["block"], st["max_blocks"]
    pb = _page_bytes(c)
    slot = ((st["table"][..., 0] - st["arena"].data_ptr()) // (2 * pb)).clamp_min(0)
    there = (st["table"][..., 2] != 0).repeat_interleave(bs, 1)
    live = there & (torch.arange(mb * bs, device="cuda")[None] < st["lens"][:, None])

    def tokens(which):                                    # [S, hkv, mb*bs, d]
        x = _pages_f32(st["arena"][:, which][slot], c)
        return x.transpose(1, 2).reshape(S, H, mb * bs, d)
    q = st["q"].float().reshape(S, H, c["hq"] // H, d)
    s = torch.matmul(q, tokens(0).transpose(2, 3)) * (1.0 / math.sqrt(d))
    s = s.masked_fill(~live[:, None, None, :], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    o = torch.matmul(p, tokens(1)) / p.sum(-1, keepdim=True).clamp_min(1e-38)
    return {"out": o.reshape(S, c["hq"], d).bfloat16()}


def _plain_layout(st):
    c = st["case"]
    n, mb, bs = c["seqs"], c["blocks"], c["block"]
    table, free = st["table"], st["free"].long()
    cap = mb * bs
    ctx = st["ctx"].long().clamp(0, cap)
    new = torch.minimum(st["new"].long().clamp_min(0), cap - ctx)
    par = st["fork"].long()
    forked = par >= 0
    p0 = par.clamp_min(0)
    ok = ~forked | ((ctx % bs == 0) & (ctx <= ctx[p0]) & (par[p0] < 0))
    ctx, new = ctx * ok, new * ok
    old, tot = (ctx + bs - 1) // bs, (ctx + new + bs - 1) // bs
    need = tot - old
    first = need.cumsum(0) - need
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), new.cumsum(0)])
    j = torch.arange(mb, device="cuda")[None]
    at = first[:, None] + j - old[:, None]
    fresh = (j >= old[:, None]) & (j < tot[:, None])
    slot = torch.where(fresh & (at < len(free)), free[at.clamp(0, len(free) - 1)], -1)
    have = (slot >= 0) & (slot < st["total"])
    addr = _BASE + slot * _SLOT_BYTES
    entry = torch.stack([(addr + _K_OFF) * have, (addr + _V_OFF) * have, have.long()], -1)
    take = forked[:, None] & (j < old[:, None])
    table.copy_(torch.where(fresh[..., None], entry,
                            torch.where(take[..., None], table[p0], table)))
    t = torch.arange(st["cap"], device="cuda")
    row = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    real = row < n
    row = row.clamp_max(n - 1)
    pos = ctx[row] + t - cu[row]
    e = table[row, (pos // bs).clamp(0, mb - 1)]
    where = torch.where(e[:, 2] != 0, (e[:, 0] - _BASE - _K_OFF) // _SLOT_BYTES * bs + pos % bs, -1)
    bad = (~ok).any() | (fresh & ~have).any() | (cu[-1] > st["cap"])
    st["err"].copy_(bad.int()[None] * 0x80)
    return {"table": table, "seq_lens": (ctx + new).int(), "cu": cu.int(),
            "token_seq": torch.where(real, row, -1).int(),
            "token_pos": torch.where(real, pos, 0).int(),
            "slot_map": torch.where(real, where, -1),
            "counts": torch.stack([cu[-1], need.sum()]).int(), "err": st["err"]}


def _plain_scores(st, logits, ranks):
    c = st["case"]
    T = torch.where(st["temperature"] > 0, st["temperature"], torch.ones_like(st["temperature"]))
    z = logits / T[:, None]
    m = z.amax(1, keepdim=True)
    dead = torch.isinf(m) & (m < 0)                       # nothing left in the row
    x = z - torch.where(dead, torch.zeros_like(m), m)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    ex = torch.where(e > 0, e * x, torch.zeros_like(x)).sum(1, keepdim=True)
    ent = torch.where(dead, torch.zeros_like(m), torch.log(total) - ex / total)
    floor = torch.where(dead, torch.zeros_like(m), lse)   # -inf - 0 where the row is dead
    tgt = st["targets"].long()
    got = {"logprob": z.gather(1, tgt) - floor, "entropy": ent[:, 0], "lse": lse[:, 0]}
    if ranks:
        lt = logits.gather(1, tgt)[..., None]
        idx = torch.arange(c["vocab"], device="cuda")[None, None]
        before = (logits[:, None] > lt) | ((logits[:, None] == lt) & (idx < tgt[..., None]))
        got["rank"] = before.sum(-1).int()
    if c["top"]:
        v, i = torch.sort(logits, dim=1, descending=True, stable=True)
        got["top_ids"] = i[:, :c["top"]].int()
        got["top_logprobs"] = v[:, :c["top"]] / T[:, None] - floor
    return got


def _plain_logprobs(st):
    return _plain_scores(st, st["logits"][:, :st["case"]["vocab"]].float(), True)


def _plain_score(st):
    return _plain_scores(st, st["hidden"].float() @ st["weight"].float().t(), False)


# ---------------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------------

_held = {}


def _backend():
    if "be" not in _held:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "xpu-kllm_b200"))
        import kllm_b200
        _held["be"] = kllm_b200.Backend()
        if _held["be"].backend != kllm_b200.KLLM_GPU_CUDA:
            raise RuntimeError("no usable device")
    return _held["be"]


def _workspace(nbytes):
    """One workspace for all calls of the program, grown when a call needs more."""
    if "ws" not in _held or _held["ws"].numel() < nbytes:
        _held["ws"] = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
    return _held["ws"].data_ptr()


def _stream():
    """torch's current stream; its default stream is the legacy one (handle 1), since a
    NULL handle selects the context's own stream."""
    return torch.cuda.current_stream().cuda_stream or 1


def _check(rc):
    if rc != 0:
        raise RuntimeError("the library refused the call: %d" % rc)


def _own_prefix(st):
    c, be = st["case"], _backend()
    nb = be.shared_prefix_workspace_size(c["seqs"], c["hq"], c["hkv"], c["d"], st["max_blocks"])
    _check(be.shared_prefix(
        output=st["out"].data_ptr(), query=st["q"].data_ptr(), block_tables=st["table"].data_ptr(),
        seq_lens=st["lens"].data_ptr(), group_starts=st["starts"].data_ptr(),
        prefix_lens=st["plens"].data_ptr(), num_seqs=c["seqs"], num_groups=c["groups"],
        num_heads=c["hq"], num_kv_heads=c["hkv"], head_dim=c["d"],
        max_blocks_per_seq=st["max_blocks"], block_size=c["block"], kv_dtype=c["kv"], layer=0,
        layer_stride=2 * _page_bytes(c), scale=1.0 / math.sqrt(c["d"]),
        workspace=_workspace(nb), workspace_bytes=nb, err_word=st["err"].data_ptr(),
        stream=_stream()))
    return {"out": st["out"]}


def _own_layout(st):
    c, be = st["case"], _backend()
    _check(be.batch_layout(
        ctx_lens=st["ctx"].data_ptr(), new_lens=st["new"].data_ptr(),
        fork_from=st["fork"].data_ptr(), free_slots=st["free"].data_ptr(),
        num_free=len(st["free"]), num_seqs=c["seqs"], max_blocks_per_seq=c["blocks"],
        block_size=c["block"], arena_base=_BASE, slot_bytes=_SLOT_BYTES, total_slots=st["total"],
        k_offset=_K_OFF, v_offset=_V_OFF, block_tables=st["table"].data_ptr(),
        seq_lens=st["seq_lens"].data_ptr(), cu_seqlens=st["cu"].data_ptr(),
        token_seq=st["token_seq"].data_ptr(), token_pos=st["token_pos"].data_ptr(),
        slot_map=st["slot_map"].data_ptr(), token_capacity=st["cap"],
        counts=st["counts"].data_ptr(), err_word=st["err"].data_ptr(), stream=_stream()))
    return {k: st[k] for k in ("table", "seq_lens", "cu", "token_seq", "token_pos", "slot_map",
                               "counts", "err")}


def _scored(st, ranks):
    got = {"logprob": st["o_lp"], "entropy": st["o_ent"], "lse": st["o_lse"]}
    if ranks:
        got["rank"] = st["o_rank"]
    if st["case"]["top"]:
        got["top_ids"], got["top_logprobs"] = st["o_ids"], st["o_top"]
    return got


def _own_logprobs(st):
    c, be = st["case"], _backend()
    _check(be.logprobs(
        logits=st["logits"].data_ptr(), logits_dtype=0 if c["dtype"] == "f32" else 1,
        row_stride=c["stride"], num_rows=c["rows"], vocab=c["vocab"],
        temperature=st["temperature"].data_ptr(), targets=st["targets"].data_ptr(),
        num_targets=c["targets"], top_n=c["top"], target_logprobs=st["o_lp"].data_ptr(),
        target_ranks=st["o_rank"].data_ptr(), entropy=st["o_ent"].data_ptr(),
        lse=st["o_lse"].data_ptr(), top_ids=st["o_ids"].data_ptr(),
        top_logprobs=st["o_top"].data_ptr(), stream=_stream()))
    return _scored(st, True)


def _own_score(st):
    c, be = st["case"], _backend()
    nb = be.score_workspace_size(c["rows"], c["vocab"], c["targets"], c["top"])
    _check(be.score_tokens(
        hidden=st["hidden"].data_ptr(), weight=st["weight"].data_ptr(), num_rows=c["rows"],
        hidden_dim=c["hidden"], vocab=c["vocab"], temperature=st["temperature"].data_ptr(),
        targets=st["targets"].data_ptr(), num_targets=c["targets"], top_n=c["top"],
        target_logprobs=st["o_lp"].data_ptr(), entropy=st["o_ent"].data_ptr(),
        lse=st["o_lse"].data_ptr(), top_ids=st["o_ids"].data_ptr(),
        top_logprobs=st["o_top"].data_ptr(), workspace=_workspace(nb), workspace_bytes=nb,
        err_word=st["err"].data_ptr(), stream=_stream()))
    return _scored(st, False)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"prefix": _own_prefix, "layout": _own_layout, "logprobs": _own_logprobs,
                "score": _own_score}[op](state)
    return {"prefix": _plain_prefix, "layout": _plain_layout, "logprobs": _plain_logprobs,
            "score": _plain_score}[op](state)


# ---------------------------------------------------------------------------------
# work and the definition in 64 bits
# ---------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "prefix":
        starts, plens, lens = _prefix_shape(c, 0)
        tok = 2 * _page_bytes(c) // c["block"]            # K and V bytes of a token
        shared = plens // c["block"] * c["block"]
        group = np.repeat(np.arange(len(plens)), np.diff(starts))
        suffix = np.maximum(0, lens - shared[group]).sum()
        rows = c["seqs"] * c["hq"] * c["d"]
        return {"bytes": int(tok * (shared.sum() + suffix) + rows * 4 + 8 * c["seqs"]),
                "flops": int(4 * c["hq"] * c["d"] * lens.sum())}
    if c["op"] == "layout":
        ctx, new, fork = _layout_shape(c, 0)
        bs = c["block"]
        old = -(-ctx // bs)
        fresh = (-(-(ctx + new) // bs) - old).sum()
        copied = (ctx // bs)[fork >= 0].sum()
        part = ((ctx % bs != 0) & (new > 0)).sum()
        return {"bytes": int(20 * c["seqs"] + 28 * fresh + 48 * copied + 24 * part
                             + 16 * _layout_capacity(c)),
                "flops": 0}
    per_row = c["targets"] * 12 + 8 + 4 + 8 * c["top"]
    if c["op"] == "logprobs":
        size = 4 if c["dtype"] == "f32" else 2
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size + c["rows"] * per_row, "flops": 6 * n}
    return {"bytes": 2 * c["hidden"] * (c["rows"] + c["vocab"]) + c["rows"] * per_row,
            "flops": 2 * c["rows"] * c["hidden"] * c["vocab"]}


def _exact_scores(st, logits):
    """From float64 logits, row by row of a chunk, by the definition."""
    c = st["case"]
    T = st["temperature"].double()
    T = torch.where(T > 0, T, torch.ones_like(T))
    z = logits / T[:, None]
    m = z.max(1).values
    dead = m == float("-inf")
    m0 = torch.where(dead, torch.zeros_like(m), m)
    p = (z - m0[:, None]).exp()
    tot = p.sum(1)
    lse = m0 + tot.log()
    p = p / tot[:, None].clamp_min(1e-300)
    ent = -torch.special.xlogy(p, p).sum(1)
    floor = torch.where(dead, torch.zeros_like(m), lse)
    got = {"logprob": z.gather(1, st["targets"].long()) - floor[:, None], "entropy": ent,
           "lse": torch.where(dead, m, lse)}
    if c["top"]:
        got["top_logprobs"] = z.topk(c["top"], 1).values - floor[:, None]
    return got


def exact(case, seed):
    if case["op"] == "layout":
        return None                                       # whole numbers only
    st = prepare(case, seed)
    c = st["case"]
    if c["op"] == "prefix":
        S, H, d, bs, pb = c["seqs"], c["hkv"], c["d"], c["block"], _page_bytes(c)
        lens = st["lens"].tolist()
        out = torch.zeros((S, c["hq"], d), dtype=torch.float64, device="cuda")
        slots = (st["table"][..., 0] - st["arena"].data_ptr()) // (2 * pb)
        for s in range(S):
            n = lens[s]
            if n == 0:
                continue
            pages = st["arena"][slots[s, :-(-n // bs)]]
            kv = _pages_f32(pages, c).double()            # an E4M3 product is exact in 32 bits
            kv = kv.permute(1, 2, 0, 3, 4).reshape(2, H, -1, d)[:, :, :n]
            q = st["q"][s].double().reshape(H, -1, d)
            w = torch.softmax(q @ kv[0].transpose(1, 2) / math.sqrt(d), -1)
            out[s] = (w @ kv[1]).reshape(c["hq"], d)
        return {"out": out}
    step = max(1, (1 << 30) // c["vocab"] // 8)
    got = []
    w = st["weight"].double().t() if c["op"] == "score" else None
    for a in range(0, c["rows"], step):
        part = dict(st, targets=st["targets"][a:a + step], temperature=st["temperature"][a:a + step])
        lg = (st["logits"][a:a + step, :c["vocab"]].double() if w is None
              else st["hidden"][a:a + step].double() @ w)
        got.append(_exact_scores(part, lg))
    both = {k: torch.cat([g[k] for g in got]) for k in got[0]}
    for k in ("rank", "top_ids"):
        if (k == "rank" and c["op"] == "logprobs") or (k == "top_ids" and c["top"]):
            both[k] = None
    return both

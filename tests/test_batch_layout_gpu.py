# SPDX-License-Identifier: Apache-2.0
"""kllm_gpu_batch_layout against its rules applied row by row on the host:
every output equal, forks, exhausted free lists, cut lengths and padding
included; and the KV append that follows takes what it lays out."""
from __future__ import annotations

import numpy as np
import pytest

import scorecase as sc
import kllm_b200 as kb

pytestmark = pytest.mark.gpu

BASE, SLOT, KO, VO = 1 << 40, 4096, 64, 2112


@pytest.fixture(scope="module")
def be():
    import torch
    b = kb.Backend()
    assert b.backend == kb.KLLM_GPU_CUDA
    torch.cuda.set_stream(b.torch_stream())
    yield b
    torch.cuda.synchronize()
    torch.cuda.set_stream(torch.cuda.default_stream())
    b.close()


def make(rng, S, mb, block, max_new, fork_every=0):
    cap = mb * block
    ctx = rng.integers(0, cap + 1, S)
    ctx[rng.random(S) < 0.2] = 0
    new = np.minimum(rng.integers(0, max_new + 1, S), cap - ctx)
    fork = np.full(S, -1)
    if fork_every:
        for s in range(1, S, fork_every):
            p = int(rng.integers(0, s))
            if fork[p] < 0:
                fork[s] = p
                ctx[s] = rng.integers(0, ctx[p] // block + 1) * block
                new[s] = min(new[s], cap - ctx[s])
    total = S * mb * 2 + 64
    slots = rng.permutation(total)
    table = np.zeros((S, mb, 3), np.int64)
    at = 0
    for s in range(S):
        for j in range(0 if fork[s] >= 0 else -(-int(ctx[s]) // block)):
            a = BASE + int(slots[at]) * SLOT
            table[s, j] = (a + KO, a + VO, 1)
            at += 1
    return ctx, new, fork, table, slots[at:], total


def run(be, ctx, new, fork, free, table, total, block, capacity, slot_map=True, counts=True,
        num_free=None, stream=None):
    import torch
    S, mb, _ = table.shape
    up = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    i = lambda *s: torch.full(s, -99, dtype=torch.int32, device="cuda")  # noqa: E731
    d = dict(ctx=up(ctx), new=up(new), fork=None if fork is None else up(fork), free=up(free))
    tb = torch.from_numpy(table.copy()).cuda()
    lens, cu, ts, tp, cn = i(max(S, 1)), i(S + 1), i(capacity + 4), i(capacity + 4), i(2)
    sm = torch.full((capacity + 4,), -99, dtype=torch.int64, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = be.batch_layout(ctx_lens=d["ctx"].data_ptr(), new_lens=d["new"].data_ptr(),
                         fork_from=None if fork is None else d["fork"].data_ptr(),
                         free_slots=d["free"].data_ptr(),
                         num_free=len(free) if num_free is None else num_free, num_seqs=S,
                         max_blocks_per_seq=mb, block_size=block, arena_base=BASE,
                         slot_bytes=SLOT, total_slots=total, k_offset=KO, v_offset=VO,
                         block_tables=tb.data_ptr(), seq_lens=lens.data_ptr(),
                         cu_seqlens=cu.data_ptr(), token_seq=ts.data_ptr(),
                         token_pos=tp.data_ptr(), slot_map=sm.data_ptr() if slot_map else None,
                         token_capacity=capacity, counts=cn.data_ptr() if counts else None,
                         err_word=err.data_ptr(),
                         stream=stream or torch.cuda.current_stream().cuda_stream)
    assert rc == 0, rc
    torch.cuda.synchronize()
    n = lambda t: t.cpu().numpy()  # noqa: E731
    for t in (ts, tp, sm):
        assert (n(t)[capacity:] == -99).all(), "written past token_capacity"
    return dict(table=n(tb), seq_lens=n(lens)[:S], cu=n(cu), token_seq=n(ts)[:capacity],
                token_pos=n(tp)[:capacity], slot_map=n(sm)[:capacity], counts=n(cn),
                err=int(err.item()))


def check(be, ctx, new, fork, free, table, total, block, capacity):
    got = run(be, ctx, new, fork, free, table, total, block, capacity)
    want = sc.layout(ctx, new, fork, free, table.copy(), block=block, base=BASE, slot_bytes=SLOT,
                     total=total, k_off=KO, v_off=VO, capacity=capacity)
    for k in want:
        assert np.array_equal(got[k], want[k]), k
    return got


@pytest.mark.parametrize("S,mb,block,max_new,fork", [
    (1, 1, 16, 1, 0), (1, 40, 16, 300, 0), (16, 8, 16, 1, 0), (33, 20, 5, 40, 3),
    (100, 30, 128, 600, 4), (1025, 12, 16, 9, 5), (4096, 6, 16, 3, 2), (300, 9, 1, 4, 3)])
def test_against_the_rules(be, S, mb, block, max_new, fork):
    rng = np.random.default_rng(S * 7 + block)
    ctx, new, fk, table, free, total = make(rng, S, mb, block, max_new, fork)
    cap = int(new.sum()) + 37
    got = check(be, ctx, new, fk if fork else None, free, table, total, block, cap)
    assert got["err"] == 0


def test_exact_capacity_and_no_padding(be):
    rng = np.random.default_rng(3)
    ctx, new, fk, table, free, total = make(rng, 50, 9, 16, 20)
    assert check(be, ctx, new, None, free, table, total, 16, int(new.sum()))["err"] == 0


def test_more_tokens_than_the_capacity(be):
    rng = np.random.default_rng(4)
    ctx, new, fk, table, free, total = make(rng, 20, 30, 16, 200)
    got = check(be, ctx, new, None, free, table, total, 16, int(new.sum()) // 2)
    assert got["err"] == kb.ERR_LAYOUT


def test_free_list_runs_out_or_names_no_slot(be):
    rng = np.random.default_rng(5)
    ctx, new, fk, table, free, total = make(rng, 12, 30, 16, 200)
    got = check(be, ctx, new, None, free[:10], table, total, 16, int(new.sum()))
    assert got["err"] == kb.ERR_LAYOUT and (got["slot_map"] == -1).any()
    free = free.copy()
    free[3], free[5] = -4, total
    got = check(be, ctx, new, None, free, table, total, 16, int(new.sum()))
    assert got["err"] == kb.ERR_LAYOUT


def test_lengths_cut_at_the_table(be):
    table = np.zeros((4, 3, 3), np.int64)
    got = check(be, [-5, 100, 40, 48], [3, 2, 20, 1], None, np.arange(20), table, 64, 16, 64)
    assert got["err"] & kb.ERR_SEQ_TOO_LONG
    assert got["seq_lens"].tolist() == [3, 48, 48, 48]


def test_forks_that_are_refused(be):
    table = np.zeros((7, 4, 3), np.int64)
    for j in range(4):
        table[0, j] = (BASE + j * SLOT + KO, BASE + j * SLOT + VO, 1)
    ctx = [50, 48, 17, 64, 16, 0, 16]
    fork = [-1, 0, 0, 0, 1, 5, 99]        # ok; half a block; beyond the parent; of a fork; itself; none
    got = check(be, ctx, [1] * 7, fork, np.arange(10, 30), table, 64, 16, 16)
    # row 3's 64 + 1 tokens are also more than its table holds
    assert got["err"] == kb.ERR_LAYOUT | kb.ERR_SEQ_TOO_LONG
    assert got["seq_lens"].tolist() == [51, 49, 0, 0, 0, 0, 0]


def test_no_rows_and_optional_outputs(be):
    got = run(be, np.zeros(1), np.zeros(1), None, np.arange(4), np.zeros((0, 2, 3), np.int64), 8,
              16, 5)
    assert got["cu"].tolist() == [0] and (got["token_seq"] == -1).all()
    rng = np.random.default_rng(6)
    ctx, new, fk, table, free, total = make(rng, 9, 9, 16, 20)
    got = run(be, ctx, new, None, free, table, total, 16, int(new.sum()) + 3, slot_map=False,
              counts=False)
    assert (got["slot_map"] == -99).all() and (got["counts"] == -99).all()
    want = sc.layout(ctx, new, None, free, table.copy(), block=16, base=BASE, slot_bytes=SLOT,
                     total=total, k_off=KO, v_off=VO, capacity=int(new.sum()) + 3)
    assert np.array_equal(got["token_pos"], want["token_pos"])


def test_refusals(be):
    import ctypes

    import torch
    t = torch.zeros(64, dtype=torch.int64, device="cuda")
    ptr = t.data_ptr()
    ok = dict(ctx_lens=ptr, new_lens=ptr, free_slots=ptr, num_free=4, num_seqs=1,
              max_blocks_per_seq=2, block_size=16, arena_base=BASE, slot_bytes=SLOT, total_slots=4,
              block_tables=ptr, seq_lens=ptr, cu_seqlens=ptr, token_seq=ptr, token_pos=ptr,
              token_capacity=1)
    bad = [(dict(flags=2), kb.EINVAL), (dict(num_seqs=-1), kb.EINVAL),
           (dict(num_seqs=4097), kb.ENOSYS), (dict(num_free=-1), kb.EINVAL),
           (dict(token_capacity=-1), kb.EINVAL), (dict(max_blocks_per_seq=0), kb.EINVAL),
           (dict(block_size=0), kb.EINVAL), (dict(slot_bytes=0), kb.EINVAL),
           (dict(max_blocks_per_seq=1 << 27, block_size=16), kb.EINVAL),
           (dict(ctx_lens=None), kb.EINVAL), (dict(new_lens=None), kb.EINVAL),
           (dict(free_slots=None), kb.EINVAL), (dict(block_tables=None), kb.EINVAL),
           (dict(block_tables=ptr + 4), kb.EINVAL), (dict(slot_map=ptr + 4), kb.EINVAL),
           (dict(seq_lens=None), kb.EINVAL), (dict(cu_seqlens=None), kb.EINVAL),
           (dict(token_seq=None), kb.EINVAL), (dict(token_pos=None), kb.EINVAL)]
    for change, code in bad:
        assert be.batch_layout(**{**ok, **change}) == code, change
    short = kb.BatchLayoutParams(struct_size=8)
    assert be.lib.kllm_gpu_batch_layout(be.ctx, ctypes.byref(short)) == kb.EINVAL


@pytest.mark.parametrize("S,mb,max_new,fork", [(4096, 8, 3, 5), (700, 40, 200, 3), (9, 20, 1, 0)])
@pytest.mark.parametrize("place", ["ctx", "new"])
def test_lengths_in_place(be, S, mb, max_new, fork, place):
    """seq_lens written over the lengths that the call reads: parents' lengths
    among them, with more token rows than one CTA would take."""
    import torch
    rng = np.random.default_rng(S + len(place))
    ctx, new, fk, table, free, total = make(rng, S, mb, 16, max_new, fork)
    capacity = int(new.sum()) + 5
    want = sc.layout(ctx, new, fk if fork else None, free, table.copy(), block=16, base=BASE,
                     slot_bytes=SLOT, total=total, k_off=KO, v_off=VO, capacity=capacity)
    up = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    d = dict(ctx=up(ctx), new=up(new), fork=up(fk), free=up(free))
    for shift in (0, 3):                     # the array itself, or one that begins inside it
        both = torch.zeros(S + shift, dtype=torch.int32, device="cuda")
        both[:S] = d[place]
        src = dict(d, **{place: both})
        lens = both[shift:]
        tb = torch.from_numpy(table.copy()).cuda()
        i = lambda n: torch.full((n,), -99, dtype=torch.int32, device="cuda")  # noqa: E731
        cu, ts, tp, cn, err = i(S + 1), i(capacity), i(capacity), i(2), i(1)
        err.zero_()
        sm = torch.zeros(capacity, dtype=torch.int64, device="cuda")
        assert be.batch_layout(
            ctx_lens=src["ctx"].data_ptr(), new_lens=src["new"].data_ptr(),
            fork_from=d["fork"].data_ptr() if fork else None, free_slots=d["free"].data_ptr(),
            num_free=len(free), num_seqs=S, max_blocks_per_seq=mb, block_size=16, arena_base=BASE,
            slot_bytes=SLOT, total_slots=total, k_offset=KO, v_offset=VO,
            block_tables=tb.data_ptr(), seq_lens=lens.data_ptr(), cu_seqlens=cu.data_ptr(),
            token_seq=ts.data_ptr(), token_pos=tp.data_ptr(), slot_map=sm.data_ptr(),
            token_capacity=capacity, counts=cn.data_ptr(), err_word=err.data_ptr(),
            stream=torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        got = dict(table=tb, seq_lens=lens, cu=cu, token_seq=ts, token_pos=tp, slot_map=sm, counts=cn)
        for k, v in got.items():
            assert np.array_equal(v.cpu().numpy(), want[k]), (k, shift)
        assert int(err.item()) == want["err"] == 0

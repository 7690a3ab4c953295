# SPDX-License-Identifier: Apache-2.0
"""kllm_gpu_shared_prefix_attention against the attention of each row over its
own table in 64 bits, and against kllm_gpu_paged_attention_v2."""
from __future__ import annotations

import ctypes
from dataclasses import replace

import numpy as np
import pytest

import prefixcase as pc
import kllm_b200 as kb
from kllm_b200 import workloads as wl

pytestmark = pytest.mark.gpu

MX, BF16 = wl.KV_MX_FP8, wl.KV_BF16


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


def cfg(kv=MX, hq=8, hkv=2, d=128, block=16, layers=1):
    return wl.DecodeConfig("shared", 1, hq, hkv, d=d, block=block, kv_dtype=kv, layers=layers)


def check(be, c, groups, err=0, **kw):
    case = pc.PrefixCase(c, groups, **kw)
    dev = pc.OnDevice(case)
    got = dev.run(be)
    assert int(dev.err.item()) == err
    pc.assert_near(got, case.want(), f"{c} {kw}")
    return case, dev, got


def suffixes(n, p, hi, seed):
    return [int(p + x) for x in np.random.default_rng(seed).integers(0, hi + 1, n)]


# one block to many; a last block that is not full; nothing but the prefix
@pytest.mark.parametrize("kv", [MX, BF16])
@pytest.mark.parametrize("prefix,hi", [(16, 0), (112, 5), (128, 40), (144, 0), (384, 17),
                                       (1000, 33), (4099, 100)])
def test_prefix_lengths(be, kv, prefix, hi):
    check(be, cfg(kv), [(prefix, suffixes(5, prefix, hi, prefix))])


# rows of a kv head from 2 to several 256-row units, odd group sizes
@pytest.mark.parametrize("kv", [MX, BF16])
@pytest.mark.parametrize("hq,hkv,n", [(2, 2, 2), (1, 1, 127), (1, 1, 129), (3, 1, 43), (8, 1, 32),
                                      (8, 1, 33), (7, 1, 90), (5, 5, 12), (6, 2, 100)])
def test_head_layouts_and_row_counts(be, kv, hq, hkv, n):
    check(be, cfg(kv, hq, hkv), [(320, suffixes(n, 320, 20, n))])


@pytest.mark.parametrize("kv", [MX, BF16])
@pytest.mark.parametrize("n", [3, 70])
def test_head_dim_64(be, kv, n):
    check(be, cfg(kv, 8, 2, d=64), [(700, suffixes(n, 700, 50, n))])


@pytest.mark.parametrize("kv", [MX, BF16])
@pytest.mark.parametrize("block", [32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_block_sizes(be, kv, block, d):
    check(be, cfg(kv, 4, 2, d=d, block=block), [(5 * block + 3, suffixes(9, 5 * block + 3, 130, 1))])


@pytest.mark.parametrize("kv", [MX, BF16])
def test_ragged_groups_and_rows_outside(be, kv):
    groups = [(500, suffixes(40, 500, 90, 1)), (33, [40]), (0, [5, 9, 0]),
              (260, suffixes(3, 260, 1, 2)), (2000, suffixes(70, 2000, 30, 3)),
              (15, [20, 30])]
    check(be, cfg(kv), groups, loose=[70, 0, 1, 300])


@pytest.mark.parametrize("kv", [MX, BF16])
def test_rows_shorter_than_the_prefix(be, kv):
    """Ended requests, and rows that left the group: each over its own table.
    The first row is one of them, so the prefix pages come from another."""
    check(be, cfg(kv), [(200, [0, 191, 260, -3, 200, 17, 192, 500])])
    check(be, cfg(kv), [(200, [0, 10, 191, 100])])       # none holds the prefix
    check(be, cfg(kv), [(64, [0, 0])], loose=[0])


def test_more_groups_than_ctas(be):
    groups = [(16 * (1 + g % 9), suffixes(2 + g % 3, 16 * (1 + g % 9), 8, g)) for g in range(170)]
    check(be, cfg(MX, 2, 2, d=64), groups)


@pytest.mark.parametrize("kv", [MX, BF16])
def test_pages_that_are_absent(be, kv):
    """Invalid entries are skipped, as in the decode: single pages, a whole
    block of 128 keys, all of the prefix; what they point to is not read."""
    c = cfg(kv)
    groups = [(700, suffixes(6, 700, 40, 5)), (128, suffixes(3, 128, 9, 6))]
    case = pc.PrefixCase(c, groups)
    case.valid[:6, [0, 3, 17, 43]] = False
    case.valid[:6, 8:16] = False
    case.valid[6:, :8] = False
    dev = pc.OnDevice(case)
    pc.assert_near(dev.run(be), case.want())


@pytest.mark.parametrize("kv", [MX, BF16])
def test_layers(be, kv):
    case = pc.PrefixCase(cfg(kv, layers=3), [(300, suffixes(5, 300, 30, 7))])
    dev = pc.OnDevice(case)
    for layer in (2, 0):
        pc.assert_near(dev.run(be, layer=layer), case.want(layer))


def test_every_payload_code(be):
    """All 256 E4M3 payload and scale codes in the prefix, 0x7F / 0xFF (+-480)
    among them."""
    case = pc.PrefixCase(cfg(MX, 4, 1), [(256, suffixes(4, 256, 0, 8))])
    sec = case.arena.reshape(len(case.arena), 2, -1)
    n = 16 * 128
    sec[:, :, :n] = np.resize(np.arange(256, dtype=np.uint8), sec[:, :, :n].shape)
    sec[:, 0, n:] = 1                        # keys of moderate size: many weigh in
    sec[:, 1, n:] = np.random.default_rng(1).integers(0, 256, sec[:, 1, n:].shape)
    dev = pc.OnDevice(case)
    pc.assert_near(dev.run(be), case.want())


@pytest.mark.parametrize("kv", [MX, BF16])
def test_large_scores_and_values(be, kv):
    """A softmax of a few keys: the reference maximum is raised many times."""
    case = pc.PrefixCase(cfg(kv), [(1500, suffixes(40, 1500, 30, 9))], magnitude=40.0)
    x = wl.bf16_to_f32(case.q)
    x[::2] *= 8
    x[5] = 0
    x[7] *= 1e-30
    case.q = wl.f32_to_bf16(x)
    dev = pc.OnDevice(case)
    pc.assert_near(dev.run(be), case.want())


@pytest.mark.parametrize("kv", [MX, BF16])
def test_agrees_with_the_decode(be, kv):
    """A serving shape: the decode of the same tables gives the same rows."""
    import torch
    c = cfg(kv, 32, 8)
    case = pc.PrefixCase(c, [(2048, suffixes(20, 2048, 200, 10))])
    dev = pc.OnDevice(case)
    got = dev.run(be)
    out = torch.zeros_like(dev.out)
    rc = be.decode_v2(output=out.data_ptr(), query=dev.q.data_ptr(),
                      block_tables=dev.tab.data_ptr(), seq_lens=dev.lens.data_ptr(), num_seqs=20,
                      num_heads=32, num_kv_heads=8, head_dim=128,
                      max_blocks_per_seq=case.max_blocks, block_size=16, kv_dtype=kv, layer=0,
                      layer_stride=c.layer_stride(), scale=c.scale, split=1,
                      stream=torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    ref = wl.bf16_to_f32(out.cpu().numpy().view(np.uint16))
    # both within the bound of the same exact value
    assert (np.abs(got - ref) <= 2 * case.want()[1]).all()


def test_groups_out_of_order_are_flagged_and_not_shared(be):
    import torch
    case = pc.PrefixCase(cfg(), [(64, suffixes(4, 64, 9, 1)), (64, suffixes(4, 64, 9, 2))])
    dev = pc.OnDevice(case)
    for starts in ([0, 6, 4], [-1, 4, 8], [0, 4, 9]):
        dev.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        pc.assert_near(dev.run(be), case.want())
        assert int(dev.err.item()) == kb.ERR_LAYOUT


def test_error_bits(be):
    case = pc.PrefixCase(cfg(), [(64, suffixes(4, 64, 9, 1))])
    dev = pc.OnDevice(case)
    dev.lens[2] = case.max_blocks * 16 + 1
    dev.run(be)
    assert int(dev.err.item()) & kb.ERR_SEQ_TOO_LONG
    # a page 8 bytes off is skipped and flagged
    case = pc.PrefixCase(cfg(), [(64, suffixes(4, 64, 9, 1))])
    dev = pc.OnDevice(case)
    t = case.table(dev.arena.data_ptr())
    t["k"][:, 1] += 8
    import torch
    dev.tab = torch.from_numpy(t.view(np.uint8).copy()).cuda()
    got = dev.run(be)
    assert int(dev.err.item()) == kb.ERR_MISALIGNED
    case.valid[:, 1] = False
    pc.assert_near(got, case.want())
    # pages outside a registered arena are skipped and flagged
    case = pc.PrefixCase(cfg(), [(64, suffixes(4, 64, 9, 1))])
    dev = pc.OnDevice(case)
    other = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    assert be.lib.kllm_gpu_register_arena(be.ctx, other.data_ptr(), 4096) == 0
    try:
        got = dev.run(be)
    finally:
        be.lib.kllm_gpu_clear_arenas(be.ctx)
    assert int(dev.err.item()) == kb.ERR_PAGE_RANGE and (got == 0).all()


@pytest.mark.parametrize("kv", [MX, BF16])
def test_more_rows_than_a_plan_keeps_at_hand(be, kv):
    """5,200 rows in 1,500 groups: the plan takes several rounds, and the tile
    sums do not fit the suffix CTAs' shared memory."""
    rng = np.random.default_rng(8)
    groups = [(16 * int(rng.integers(0, 3)) + 3, rng.integers(0, 70, 3).tolist()) for _ in range(1500)]
    check(be, cfg(kv, 2, 1, d=64), groups, loose=rng.integers(0, 40, 700).tolist())


def test_same_bits_every_time_and_on_another_stream(be):
    import torch
    case = pc.PrefixCase(cfg(MX, 32, 8), [(1111, suffixes(30, 1111, 60, 3))])
    dev = pc.OnDevice(case)
    a = dev.run(be)
    assert (a == dev.run(be)).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert (a == dev.run(be, stream=side.cuda_stream)).all()


def test_capture_in_a_graph(be):
    import torch
    case = pc.PrefixCase(cfg(), [(300, suffixes(6, 300, 30, 4))])
    dev = pc.OnDevice(case)
    want = dev.run(be)
    nb = be.shared_prefix_workspace_size(6, 8, 2, 128, case.max_blocks)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    dev.out.fill_(0x7FC0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rc = be.shared_prefix(**dev.kwargs(workspace=ws.data_ptr(), workspace_bytes=nb,
                                           stream=torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    g.replay()
    torch.cuda.synchronize()
    assert (wl.bf16_to_f32(dev.out.cpu().numpy().view(np.uint16)) == want).all()


def test_traced_as_its_own_operation(be):
    import torch
    case = pc.PrefixCase(cfg(), [(64, suffixes(4, 64, 9, 1))])
    dev = pc.OnDevice(case)
    assert be.lib.kllm_gpu_trace_enable(be.ctx, 8) == 0
    try:
        dev.run(be)
        torch.cuda.synchronize()
        rec = (kb.TraceRecord * 4)()
        dropped = ctypes.c_uint64()
        assert be.lib.kllm_gpu_trace_read(be.ctx, rec, 4, ctypes.byref(dropped)) == 1
        assert rec[0].op == kb.TRACE_SHARED and rec[0].gpu_us > 0
    finally:
        be.lib.kllm_gpu_trace_enable(be.ctx, 0)


def test_refusals(be):
    import torch
    case = pc.PrefixCase(cfg(), [(64, suffixes(4, 64, 9, 1))])
    dev = pc.OnDevice(case)
    nb = be.shared_prefix_workspace_size(4, 8, 2, 128, case.max_blocks)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    ok = dev.kwargs(workspace=ws.data_ptr(), workspace_bytes=nb)
    bad = [(dict(flags=1), kb.EINVAL), (dict(output=None), kb.EINVAL), (dict(query=None), kb.EINVAL),
           (dict(block_tables=None), kb.EINVAL), (dict(seq_lens=None), kb.EINVAL),
           (dict(group_starts=None), kb.EINVAL), (dict(prefix_lens=None), kb.EINVAL),
           (dict(num_groups=-1), kb.EINVAL), (dict(num_groups=5), kb.EINVAL),
           (dict(num_seqs=-1), kb.EINVAL), (dict(num_heads=7), kb.EINVAL),
           (dict(num_heads=18), kb.ENOSYS), (dict(head_dim=96), kb.ENOSYS),
           (dict(block_size=24), kb.ENOSYS), (dict(block_size=144), kb.ENOSYS),
           (dict(kv_dtype=2), kb.ENOSYS), (dict(layer=-1), kb.EINVAL),
           (dict(layer_stride=8), kb.EINVAL), (dict(max_blocks_per_seq=0), kb.EINVAL),
           (dict(query=dev.q.data_ptr() + 2), kb.EINVAL), (dict(workspace=None), kb.EINVAL),
           (dict(workspace=ws.data_ptr() + 8), kb.EINVAL), (dict(workspace_bytes=nb - 1), kb.ENOSPC)]
    for change, code in bad:
        assert be.shared_prefix(**{**ok, **change}) == code, change
    assert be.shared_prefix(**{**ok, "num_seqs": 0, "num_groups": 0}) == 0
    short = kb.SharedPrefixParams(struct_size=8)
    assert be.lib.kllm_gpu_shared_prefix_attention(be.ctx, ctypes.byref(short)) == kb.EINVAL


def decode_of(be, case, dev, scale):
    """kllm_gpu_paged_attention_v2 of the same tables."""
    import torch
    c = case.cfg
    out = torch.zeros_like(dev.out)
    rc = be.decode_v2(output=out.data_ptr(), query=dev.q.data_ptr(),
                      block_tables=dev.tab.data_ptr(), seq_lens=dev.lens.data_ptr(),
                      num_seqs=len(case.lens), num_heads=c.hq, num_kv_heads=c.hkv, head_dim=c.d,
                      max_blocks_per_seq=case.max_blocks, block_size=c.block, kv_dtype=c.kv_dtype,
                      layer=0, layer_stride=c.layer_stride(), scale=scale, split=1,
                      stream=torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    return wl.bf16_to_f32(out.cpu().numpy().view(np.uint16))


def assert_contract(got, want, what):
    """The parity contract of attention outputs."""
    r = np.abs(got - want) / (1e-3 + 2e-2 * np.abs(want))
    assert np.isfinite(got).all() and r.max() <= 1.0, (what, float(r.max()))


@pytest.mark.parametrize("kv,size,unit", [(MX, 4000.0, 1 / 64), (BF16, 400.0, 1 / 16)])
@pytest.mark.parametrize("hq,hkv,n", [(8, 2, 6), (8, 1, 33)])
def test_values_that_cancel(be, kv, size, unit, hq, hkv, n):
    """Two keys of nearly equal weight hold nearly opposite values: the output
    is what is left of a few thousand, so P has to keep more bits than the
    output. The two lie in one block, or in blocks of different streams."""
    import kvcase
    import oracle
    c = cfg(kv, hq, hkv)
    rng = np.random.default_rng(n)
    for first, second in ((37, 90), (37, 200), (130, 390)):
        case = pc.PrefixCase(c, [(400, suffixes(n, 400, 20, 3))])
        pages, bs = len(case.arena), c.block
        k = np.zeros((pages * bs, hkv, c.d), np.float32)
        v = rng.standard_normal(k.shape).astype(np.float32)
        amp = size * (0.25 + 0.75 * rng.random((hkv, c.d)))
        for tok, sign in ((first, 1.0), (second, -1.0)):
            at = case.slots[0, tok // bs] * bs + tok % bs
            k[at], k[at, :, 0] = 8.0, sign / 16           # 20 nats above the others
            v[at] = sign * amp
        for which, x in ((0, k), (1, v)):
            b = wl.f32_to_bf16(x)
            pay, sc = oracle.mx_quantize(b) if kv == MX else (b, None)
            case.arena[:, 0, which] = kvcase._pages_from_rows(c, pay, sc, pages, 0)
        q = np.full((n, hq, c.d), 0.25, np.float32)
        q[:, :, 0] = rng.integers(4, 30, (n, hq)) * unit * rng.choice([-1, 1], (n, hq))
        case.q = wl.f32_to_bf16(q)
        dev = pc.OnDevice(case)
        want = case.want()[0]
        assert np.median(np.abs(want)) > 0.3
        assert_contract(decode_of(be, case, dev, c.scale), want, "decode")
        assert_contract(dev.run(be), want, (first, second))


@pytest.mark.parametrize("kv", [MX, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.02, -0.0884])
def test_scales_of_zero_and_below(be, kv, scale):
    """As the decode has them: equal weights, or the smallest products first.
    Blocks that are not full, absent pages, one query tile and two."""
    class Scaled(wl.DecodeConfig):
        @property
        def scale(self):
            return scale
    for hq, hkv, n, p in ((8, 2, 5, 200), (8, 1, 33, 400), (4, 4, 3, 128)):
        c = Scaled("shared", 1, hq, hkv, kv_dtype=kv)
        case = pc.PrefixCase(c, [(p, suffixes(n, p, 30, 2))])
        case.valid[:, [1, 6]] = False
        dev = pc.OnDevice(case)
        want = case.want()[0]
        assert_contract(decode_of(be, case, dev, scale), want, "decode")
        assert_contract(dev.run(be), want, (hq, hkv, n, p))


@pytest.mark.parametrize("kv", [MX, BF16])
def test_rows_that_hold_the_whole_pages_only(be, kv):
    """A row of 192 to 199 tokens does not hold a prefix of 200, so its pages
    are its own, the first row's among them."""
    case = pc.PrefixCase(cfg(kv), [(200, [195, 260, 192, 200, 199, 300])], loose=[195, 192, 199])
    for row, other in ((0, 6), (2, 7), (4, 8)):
        case.slots[row] = case.slots[other]
    dev = pc.OnDevice(case)
    pc.assert_near(dev.run(be), case.want())
    case = pc.PrefixCase(cfg(kv), [(200, [195, 199])], loose=[195, 199])     # and no row that does
    case.slots[0], case.slots[1] = case.slots[2], case.slots[3]
    dev = pc.OnDevice(case)
    pc.assert_near(dev.run(be), case.want())

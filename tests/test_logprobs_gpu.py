# SPDX-License-Identifier: Apache-2.0
"""kllm_gpu_logprobs against the definition in 64 bits: log-probabilities and
entropy within the bound of their fp32 sums, ranks and top alternatives equal,
ties, masks, NaN, infinities, strides and misaligned rows included."""
from __future__ import annotations

import numpy as np
import pytest

import scorecase as sc
import kllm_b200 as kb
from kllm_b200 import workloads as wl

pytestmark = pytest.mark.gpu


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


def run(be, logits, targets, top_n, temperature=None, bf16=False, pad=0, shift=0, stream=None):
    """logits float32 [R, V] (bf16 values when bf16). pad: elements between
    rows; shift: elements the first row starts after an aligned address."""
    import torch
    R, V = logits.shape
    x = wl.f32_to_bf16(logits).view(np.int16) if bf16 else logits.astype(np.float32)
    poison = np.int16(0x7fc0) if bf16 else np.float32(np.nan)      # NaN outside the rows
    buf = np.full(shift + R * (V + pad) + 16, poison, x.dtype)
    for r in range(R):
        a = shift + r * (V + pad)
        buf[a:a + V] = x[r]
    dev = torch.from_numpy(buf).cuda()
    nt = targets.shape[1]
    tgt = torch.from_numpy(targets.astype(np.int32)).cuda()
    tmp = None if temperature is None else torch.from_numpy(
        np.asarray(temperature, np.float32)).cuda()
    f = lambda *s: torch.full(s, 7.5, dtype=torch.float32, device="cuda")  # noqa: E731
    i = lambda *s: torch.full(s, -77, dtype=torch.int32, device="cuda")  # noqa: E731
    lp, rk, en, ls = f(R, max(nt, 1)), i(R, max(nt, 1)), f(R), f(R)
    ids, tlp = i(R, max(top_n, 1)), f(R, max(top_n, 1))
    rc = be.logprobs(logits=dev.data_ptr() + shift * buf.itemsize,
                     logits_dtype=kb.LOGITS_BF16 if bf16 else kb.LOGITS_F32, num_rows=R,
                     row_stride=V + pad, vocab=V, num_targets=nt,
                     temperature=None if tmp is None else tmp.data_ptr(),
                     targets=tgt.data_ptr(), target_logprobs=lp.data_ptr(),
                     target_ranks=rk.data_ptr(), entropy=en.data_ptr(), lse=ls.data_ptr(),
                     top_n=top_n, top_ids=ids.data_ptr(), top_logprobs=tlp.data_ptr(),
                     stream=stream or torch.cuda.current_stream().cuda_stream)
    assert rc == 0, (rc, be.stats().last_cuda_error)
    torch.cuda.synchronize()
    n = lambda t: t.cpu().numpy()  # noqa: E731
    return dict(logprob=n(lp)[:, :nt], rank=n(rk)[:, :nt], entropy=n(en), lse=n(ls),
                top_ids=n(ids)[:, :top_n], top_logprobs=n(tlp)[:, :top_n])


def check(be, logits, targets, top_n, temperature=None, bf16=False, **kw):
    if bf16:
        logits = wl.bf16_to_f32(wl.f32_to_bf16(logits))
    got = run(be, logits, targets, top_n, temperature, bf16, **kw)
    want = sc.rows(logits, temperature, targets, top_n)
    tl, te = sc.bounds(want, logits.shape[1])
    sc.assert_near(got["lse"], want["lse"], tl, "lse")
    sc.assert_near(got["entropy"], want["entropy"], te, "entropy")
    sc.assert_near(got["logprob"], want["logprob"], tl[:, None], "logprob")
    sc.assert_near(got["top_logprobs"], want["top_logprobs"], tl[:, None], "top_logprobs")
    assert (got["rank"] == want["rank"]).all()
    assert (got["top_ids"] == want["top_ids"]).all()
    return got


def normal(R, V, seed, scale=3.0):
    return (np.random.default_rng(seed).standard_normal((R, V)) * scale).astype(np.float32)


def some_targets(R, V, nt, seed):
    return np.random.default_rng(seed + 99).integers(0, V, (R, nt))


# one row spread over eight CTAs, several clusters sizes, more rows than SMs
@pytest.mark.parametrize("R,V", [(1, 128256), (3, 32003), (40, 20000), (80, 17000), (301, 5000),
                                 (2, 4095), (5, 257), (3, 33), (7, 1), (1, 300000)])
@pytest.mark.parametrize("bf16", [False, True])
def test_shapes(be, R, V, bf16):
    nt = min(3, V)
    check(be, normal(R, V, R + V), some_targets(R, V, nt, V), min(20, V),
          temperature=np.linspace(0.4, 1.6, R), bf16=bf16)


@pytest.mark.parametrize("nt,top", [(0, 32), (0, 1), (1, 0), (8, 0), (0, 0), (2, 5)])
def test_counts(be, nt, top):
    check(be, normal(4, 9001, nt * 40 + top), some_targets(4, 9001, nt, top), top)


@pytest.mark.parametrize("shift,pad", [(0, 1), (1, 0), (3, 13), (7, 5), (2, 2)])
@pytest.mark.parametrize("bf16", [False, True])
def test_strides_and_misaligned_rows(be, shift, pad, bf16):
    x = normal(5, 8191, shift * 10 + pad)
    x[1, :4] = -np.inf                      # the padding before a row reads as -inf too
    t = some_targets(5, 8191, 2, 1)
    t[1] = (3, 0)
    check(be, x, t, 20, bf16=bf16, shift=shift, pad=pad)


@pytest.mark.parametrize("V", [700, 33000])
def test_equal_logits_take_the_lowest_index(be, V):
    x = np.zeros((4, V), np.float32)
    x[1, V // 2:] = 1.0                     # half the row tied at the top
    x[2] = np.round(normal(1, V, 3)[0])     # a few dozen values only
    x[3, ::7] = -0.0                        # equal to +0
    check(be, x, np.tile([0, V // 2, V - 1], (4, 1)), 32)


def test_masked_rows(be):
    V = 50001
    x = normal(7, V, 5)
    x[0] = -np.inf                          # a mask that leaves nothing
    x[1] = -np.inf
    x[1, 40000] = 2.0                       # one token left
    x[2, 200:] = -np.inf                    # fewer segments than alternatives
    x[3, :-3] = -np.inf
    x[4] = np.finfo(np.float32).min         # masks of the type's lowest value
    x[4, 77] = 1.0
    x[5, 1::2] = -np.inf
    check(be, x, np.tile([0, 77, 40000, V - 1], (7, 1)), 20,
          temperature=[1, 1, 0.5, 2, 1, 0.7, 1])


def test_nan_and_infinity(be):
    V = 20011
    x = normal(4, V, 6)
    x[0, 12345] = np.nan
    x[1, 5] = np.inf
    x[2] = np.nan
    got = check(be, x, np.tile([5, 12345, 19000], (4, 1)), 20)
    assert np.isnan(got["lse"][:3]).all() and np.isfinite(got["lse"][3])


def test_targets_outside_the_vocabulary(be):
    x = normal(2, 4100, 8)
    t = np.array([[-1, 4100, 5], [2 ** 31 - 1, -2 ** 31, 4099]])
    got = check(be, x, t, 3)
    assert (got["rank"][:, :2] == -1).all() and np.isneginf(got["logprob"][:, :2]).all()


def test_large_and_small_values(be):
    x = normal(3, 30000, 9)
    x[0] *= 1000.0
    x[1] *= 1e-6
    x[2] = x[2] * 1e-3 + 5e4
    check(be, x, some_targets(3, 30000, 2, 3), 20, temperature=[1.0, 0.0, -1.0])


def test_row_offsets_past_32_bits(be):
    """Rows 2^30 elements apart: the last starts past 4 GiB of bf16 logits."""
    import torch
    V, R, stride = 5000, 3, 1 << 30
    buf = torch.empty((R - 1) * stride + V, dtype=torch.bfloat16, device="cuda")
    x = wl.bf16_to_f32(wl.f32_to_bf16(normal(R, V, 11)))
    for r in range(R):
        buf[r * stride:r * stride + V] = torch.from_numpy(x[r]).cuda().bfloat16()
    lse = torch.zeros(R, device="cuda")
    ids = torch.zeros((R, 4), dtype=torch.int32, device="cuda")
    top = torch.zeros((R, 4), device="cuda")
    rc = be.logprobs(logits=buf.data_ptr(), logits_dtype=kb.LOGITS_BF16, num_rows=R,
                     row_stride=stride, vocab=V, num_targets=0, lse=lse.data_ptr(), top_n=4,
                     top_ids=ids.data_ptr(), top_logprobs=top.data_ptr(),
                     stream=torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    want = sc.rows(x, None, np.zeros((R, 0), int), 4)
    assert (ids.cpu().numpy() == want["top_ids"]).all()
    sc.assert_near(lse.cpu().numpy(), want["lse"], sc.bounds(want, V)[0], "lse")


def test_same_bits_every_time_and_on_another_stream(be):
    import torch
    x, t = normal(9, 128256, 12), some_targets(9, 128256, 2, 4)
    a = run(be, x, t, 20)
    side = torch.cuda.Stream()
    b = run(be, x, t, 20, stream=side.cuda_stream)
    for k in a:
        assert np.array_equal(a[k], b[k]), k


def test_refusals(be):
    import torch
    x = torch.zeros((2, 64), device="cuda")
    t = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    f = torch.zeros((2, 32), device="cuda")
    ok = dict(logits=x.data_ptr(), num_rows=2, vocab=64, num_targets=1, targets=t.data_ptr(),
              target_logprobs=f.data_ptr(), top_n=2, top_ids=t.data_ptr(),
              top_logprobs=f.data_ptr())
    bad = [(dict(flags=1), kb.EINVAL), (dict(logits=None), kb.EINVAL),
           (dict(logits=x.data_ptr() + 2), kb.EINVAL), (dict(vocab=0), kb.EINVAL),
           (dict(num_rows=-1), kb.EINVAL), (dict(row_stride=63), kb.EINVAL),
           (dict(num_targets=-1), kb.EINVAL), (dict(num_targets=9), kb.ENOSYS),
           (dict(targets=None), kb.EINVAL), (dict(target_logprobs=None), kb.EINVAL),
           (dict(top_n=33), kb.ENOSYS), (dict(top_n=-1), kb.EINVAL),
           (dict(top_n=5, vocab=4), kb.EINVAL), (dict(top_ids=None), kb.EINVAL),
           (dict(top_logprobs=None), kb.EINVAL), (dict(logits_dtype=2), kb.ENOSYS)]
    for change, code in bad:
        assert be.logprobs(**{**ok, **change}) == code, change
    assert be.logprobs(**{**ok, "num_rows": 0}) == 0
    short = kb.LogprobsParams(struct_size=8)
    import ctypes
    assert be.lib.kllm_gpu_logprobs(be.ctx, ctypes.byref(short)) == kb.EINVAL


@pytest.mark.parametrize("bf16", [False, True])
def test_a_vocabulary_past_the_segment_table(be, bf16):
    """More than 1,024 segments of four vectors: segments grow with the row."""
    V = 1300007
    check(be, normal(2, V, 21), some_targets(2, V, 3, 5), 32, bf16=bf16, shift=1)


@pytest.mark.parametrize("R,V", [(2, 128256), (300, 70001), (3, 33000), (400, 5000)])
@pytest.mark.parametrize("bf16", [False, True])
def test_finite_masks_with_few_tokens_allowed(be, R, V, bf16):
    """Thousands of equal logits under a handful of larger ones that lie far
    apart: the exact selection meets one of those in every part of the row.
    Fewer and more of them than alternatives; rows of one CTA and of several."""
    fills = [-1e4, -3.0, -1e4, 0.0]          # bf16 values or nearly so
    x = np.empty((R, V), np.float32)
    t = np.zeros((R, 2), int)
    for r in range(R):
        n = 2 + 3 * (r % 4)                  # 2 .. 11 allowed tokens
        at = (np.arange(n) * (V - 2)) // (n - 1) + (r % 2)
        x[r] = fills[r % 4]
        x[r, at] = 1.0 + np.arange(n) % 5
        t[r] = (at[-1], at[0] + 1)
    check(be, x, t, 7 if R > 100 else 20, bf16=bf16)


@pytest.mark.parametrize("R,V", [(1, 128256), (3, 33000), (5, 700)])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("temperature", [None, 4.0, 0.5])
def test_rows_of_the_lowest_value(be, R, V, bf16, temperature):
    """A finite mask that leaves nothing is a row of equal logits: its softmax
    is uniform. The largest finite logits, and both in one row, hold as well."""
    import torch
    low = float(torch.finfo(torch.bfloat16 if bf16 else torch.float32).min)
    t = np.tile([0, V // 2, V - 1], (R, 1))
    tmp = None if temperature is None else np.full(R, temperature, np.float32)
    for fill, other in ((low, low), (-low, -low), (low, -low)):
        x = np.full((R, V), fill, np.float32)
        x[:, 1::3] = other
        got = run(be, x, t, 20, tmp, bf16)
        n = V if fill == other else len(range(1, V, 3))
        tol = sc.distance_bound(np.log(n), 0.0, V)
        sc.assert_near(got["entropy"], np.full(R, np.log(n)), 4 * tol, "entropy")
        sc.assert_near(got["top_logprobs"], np.full((R, 20), -np.log(n)), tol, "top")
        want = np.where(x[np.arange(R)[:, None], t] == x.max(1, keepdims=True), -np.log(n), -np.inf)
        lp = got["logprob"].astype(np.float64)
        lp = np.where(lp < -1e30, -np.inf, lp)      # a distance of 6.8e38 / T rounds to -inf or not
        sc.assert_near(lp, want, tol, "logprob")
        first = np.arange(20) if fill == other else 1 + 3 * np.arange(20)
        assert (got["top_ids"] == first).all()
        with np.errstate(over="ignore"):
            lse = (np.float64(max(fill, other)) / (temperature or 1.0) + np.log(n)).astype(np.float32)
        fine = np.where(np.isfinite(lse), 2.0 ** -20 * np.abs(lse), 0.0)
        sc.assert_near(got["lse"], np.full(R, lse, np.float64), fine, "lse")


@pytest.mark.parametrize("offset,temperature", [(0, None), (1000, None), (-5e4, None), (0, 0.01),
                                                (0, 1e-3), (300, 0.02), (-1e6, 0.5)])
@pytest.mark.parametrize("R,V", [(1, 128256), (40, 20000), (5, 3001)])
def test_distances_to_the_maximum(be, R, V, offset, temperature):
    """Log-probabilities depend on the distance to the row's maximum alone: a
    common offset and a low temperature cost no accuracy, and none is above 0."""
    x = normal(R, V, V + R) + np.float32(offset)
    tmp = None if temperature is None else np.full(R, temperature, np.float32)
    t = some_targets(R, V, 3, 8)
    t[:, 2] = x.argmax(1)
    got = run(be, x, t, 20, tmp)
    sc.assert_distances(got, sc.rows(x, tmp, t, 20), V)

# SPDX-License-Identifier: Apache-2.0
"""kllm_gpu_score_tokens against the definition in 64 bits. Hidden states and
weights on a grid of powers of two make every logit exact in fp32 whatever the
order of its sum, so that the top alternatives have to be equal; a case with
ordinary values holds the numbers to the bound of the fp32 sums."""
from __future__ import annotations

import ctypes

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


def grid_case(R, K, V, seed):
    rng = np.random.default_rng(seed)
    h = np.clip(np.round(rng.standard_normal((R, K)) * 8), -32, 32) / 4
    w = np.clip(np.round(rng.standard_normal((V, K)) * 10 * np.sqrt(4096 / K)), -127, 127) / 512
    return h.astype(np.float32), w.astype(np.float32)


def run(be, h, w, targets, top_n, temperature=None, stream=None, slack=0):
    import torch
    R, K = h.shape
    V, nt = w.shape[0], targets.shape[1]
    dh = torch.from_numpy(wl.f32_to_bf16(h).view(np.int16)).cuda()
    dw = torch.from_numpy(wl.f32_to_bf16(w).view(np.int16)).cuda()
    tgt = torch.from_numpy(targets.astype(np.int32)).cuda()
    tmp = None if temperature is None else torch.from_numpy(
        np.asarray(temperature, np.float32)).cuda()
    f = lambda *s: torch.full(s, 7.5, dtype=torch.float32, device="cuda")  # noqa: E731
    lp, en, ls, tlp = f(R, max(nt, 1)), f(R), f(R), f(R, max(top_n, 1))
    ids = torch.full((R, max(top_n, 1)), -77, dtype=torch.int32, device="cuda")
    nb = be.score_workspace_size(R, V, nt, top_n)
    assert nb > 0
    ws = torch.full((nb + 64,), 0xA5, dtype=torch.uint8, device="cuda")    # no set-up needed
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = be.score_tokens(hidden=dh.data_ptr(), weight=dw.data_ptr(), num_rows=R, hidden_dim=K,
                         vocab=V, num_targets=nt,
                         temperature=None if tmp is None else tmp.data_ptr(),
                         targets=tgt.data_ptr(), target_logprobs=lp.data_ptr(),
                         entropy=en.data_ptr(), lse=ls.data_ptr(), top_n=top_n,
                         top_ids=ids.data_ptr(), top_logprobs=tlp.data_ptr(),
                         workspace=ws.data_ptr(), workspace_bytes=nb, err_word=err.data_ptr(),
                         stream=stream or torch.cuda.current_stream().cuda_stream)
    assert rc == 0, (rc, be.stats().last_cuda_error)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert (ws[nb:] == 0xA5).all(), "written past the workspace"
    n = lambda t: t.cpu().numpy()  # noqa: E731
    return dict(logprob=n(lp)[:, :nt], entropy=n(en), lse=n(ls), top_ids=n(ids)[:, :top_n],
                top_logprobs=n(tlp)[:, :top_n])


def check(be, h, w, targets, top_n, temperature=None, logit_err=0.0, ids=True):
    got = run(be, h, w, targets, top_n, temperature)
    logits = h.astype(np.float64) @ w.astype(np.float64).T
    want = sc.rows(logits, temperature, targets, top_n)
    tl, te = sc.bounds(want, w.shape[0])
    tl, te = tl + logit_err, te + logit_err * (2 + np.log(w.shape[0]))
    sc.assert_near(got["lse"], want["lse"], tl, "lse")
    sc.assert_near(got["entropy"], want["entropy"], te, "entropy")
    sc.assert_near(got["logprob"], want["logprob"], tl[:, None], "logprob")
    sc.assert_near(got["top_logprobs"], want["top_logprobs"], tl[:, None], "top_logprobs")
    if ids:
        assert (got["top_ids"] == want["top_ids"]).all()
    return got


def some_targets(R, V, nt, seed):
    return np.random.default_rng(seed + 99).integers(0, V, (R, nt))


@pytest.mark.parametrize("R,K,V,nt,top", [
    (1, 64, 1, 1, 1), (1, 64, 40, 2, 32), (3, 128, 63, 1, 20), (17, 256, 4097, 3, 20),
    (128, 64, 9000, 1, 5), (129, 192, 9001, 1, 32), (333, 1024, 3203, 1, 20),
    (257, 64, 40000, 0, 20), (2100, 64, 2000, 1, 3), (1, 4096, 32003, 8, 20), (40, 64, 257, 1, 0),
    (700, 128, 130, 2, 32)])
def test_shapes(be, R, K, V, nt, top):
    h, w = grid_case(R, K, V, R * 3 + V)
    check(be, h, w, some_targets(R, V, nt, V), top, temperature=np.linspace(0.5, 1.5, R))


@pytest.mark.parametrize("V", [1000, 33000])
def test_equal_logits_take_the_lowest_index(be, V):
    R, K = 5, 64
    h, w = grid_case(R, K, V, 7)
    h[1] = 0                                 # every logit 0
    w[:] = w[np.arange(V) % 13]              # thirteen different logits a row
    h[2] = 0
    h[2, 0] = 0.25
    w[V // 3:, 0] = 0.125                    # two thirds of row 2 tied at the top
    check(be, h, w, some_targets(R, V, 2, 1), 32)


def test_ascending_logits_replace_the_whole_list(be):
    V, K = 20000, 64
    h = np.zeros((2, K), np.float32)
    w = np.zeros((V, K), np.float32)
    h[:, 0], h[:, 1] = 8.0, 1.0 / 16
    w[:, 0] = np.arange(V) // 128 / 4.0      # bf16 values: coarse and fine parts
    w[:, 1] = np.arange(V) % 128 / 2.0
    h[1] = -h[1]                             # and descending
    check(be, h, w, some_targets(2, V, 1, 2), 32)


def test_ordinary_values(be):
    rng = np.random.default_rng(5)
    R, K, V = 200, 2048, 20011
    h = wl.bf16_to_f32(wl.f32_to_bf16(rng.standard_normal((R, K)).astype(np.float32)))
    w = wl.bf16_to_f32(wl.f32_to_bf16((rng.standard_normal((V, K)) * 0.05).astype(np.float32)))
    # fp32 sums of K products, any order: K eps sum |h w|
    err = K * sc.EPS * (np.abs(h).astype(np.float64) @ np.abs(w).T.astype(np.float64)).max(1)
    check(be, h, w, some_targets(R, V, 2, 3), 20, temperature=np.full(R, 0.8), logit_err=err / 0.8,
          ids=False)


def test_nan_infinite_and_outside_targets(be):
    R, K, V = 4, 64, 2000
    h, w = grid_case(R, K, V, 9)
    h[0, 3] = np.nan
    t = np.array([[1, 2]] * R)
    t[2] = (-1, V)
    got = run(be, h, w, t, 20)
    assert np.isnan(got["lse"][0]) and np.isnan(got["logprob"][0]).all()
    assert (got["top_ids"][0] == -1).all() and np.isneginf(got["top_logprobs"][0]).all()
    assert np.isneginf(got["logprob"][2]).all() and np.isfinite(got["lse"][1:]).all()
    want = sc.rows(h[1:].astype(np.float64) @ w.T, None, t[1:], 20)
    assert (got["top_ids"][1:] == want["top_ids"]).all()


def test_same_bits_every_time_and_on_another_stream(be):
    import torch
    h, w = grid_case(300, 256, 32003, 12)
    t = some_targets(300, 32003, 1, 4)
    a = run(be, h, w, t, 20)
    b = run(be, h, w, t, 20, stream=torch.cuda.Stream().cuda_stream)
    for k in a:
        assert np.array_equal(a[k], b[k]), k


def test_agrees_with_the_logits_path(be):
    """lm_head writes the logits, kllm_gpu_logprobs reads them: the same numbers."""
    import torch
    R, K, V = 64, 512, 8192
    h, w = grid_case(R, K, V, 13)
    t = some_targets(R, V, 1, 5)
    a = run(be, h, w, t, 20)
    dh = torch.from_numpy(wl.f32_to_bf16(h).view(np.int16)).cuda()
    dw = torch.from_numpy(wl.f32_to_bf16(w).view(np.int16)).cuda()
    logits = torch.zeros((R, V), device="cuda")
    tok = torch.zeros(R, dtype=torch.int32, device="cuda")
    ws = torch.zeros(be.lib.kllm_gpu_lm_head_workspace_size(R, V), dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    assert be.lm_head(hidden=dh.data_ptr(), weight=dw.data_ptr(), num_rows=R, hidden_dim=K,
                      vocab=V, logits=logits.data_ptr(), tokens=tok.data_ptr(),
                      workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=st) == 0
    dt = torch.from_numpy(t.astype(np.int32)).cuda()
    lp, lse, top = (torch.zeros(s, device="cuda") for s in ((R, 1), (R,), (R, 20)))
    ids = torch.zeros((R, 20), dtype=torch.int32, device="cuda")
    assert be.logprobs(logits=logits.data_ptr(), num_rows=R, vocab=V, num_targets=1,
                       targets=dt.data_ptr(), target_logprobs=lp.data_ptr(), lse=lse.data_ptr(),
                       top_n=20, top_ids=ids.data_ptr(), top_logprobs=top.data_ptr(),
                       stream=st) == 0
    torch.cuda.synchronize()
    assert (ids.cpu().numpy() == a["top_ids"]).all()
    assert (ids.cpu().numpy()[:, 0] == tok.cpu().numpy()).all()
    want = sc.rows(h.astype(np.float64) @ w.T, None, t, 20)
    tol = 2 * sc.bounds(want, V)[0]
    sc.assert_near(a["lse"], lse.cpu().numpy(), tol, "lse")
    sc.assert_near(a["logprob"], lp.cpu().numpy(), tol[:, None], "logprob")


def test_refusals(be):
    import torch
    x = torch.zeros(4096, device="cuda")
    ptr = x.data_ptr()
    nb = be.score_workspace_size(2, 64, 1, 2)
    ws = torch.zeros(nb, dtype=torch.uint8, device="cuda")
    ok = dict(hidden=ptr, weight=ptr, num_rows=2, hidden_dim=64, vocab=64, num_targets=1,
              targets=ptr, target_logprobs=ptr, top_n=2, top_ids=ptr, top_logprobs=ptr,
              workspace=ws.data_ptr(), workspace_bytes=nb)
    bad = [(dict(flags=1), kb.EINVAL), (dict(hidden=None), kb.EINVAL),
           (dict(weight=None), kb.EINVAL), (dict(hidden=ptr + 8), kb.EINVAL),
           (dict(weight=ptr + 2), kb.EINVAL), (dict(num_rows=-1), kb.EINVAL),
           (dict(num_rows=(1 << 20) + 1), kb.ENOSYS), (dict(hidden_dim=0), kb.EINVAL),
           (dict(hidden_dim=96), kb.ENOSYS), (dict(vocab=0), kb.EINVAL),
           (dict(num_targets=9), kb.ENOSYS), (dict(num_targets=-1), kb.EINVAL),
           (dict(targets=None), kb.EINVAL), (dict(target_logprobs=None), kb.EINVAL),
           (dict(top_n=33), kb.ENOSYS), (dict(top_n=65, vocab=64), kb.EINVAL),
           (dict(top_ids=None), kb.EINVAL), (dict(top_logprobs=None), kb.EINVAL),
           (dict(workspace=None), kb.EINVAL), (dict(workspace=ws.data_ptr() + 4), kb.EINVAL),
           (dict(workspace_bytes=nb - 1), kb.ENOSPC)]
    for change, code in bad:
        assert be.score_tokens(**{**ok, **change}) == code, change
    assert be.score_tokens(**{**ok, "num_rows": 0}) == 0
    short = kb.ScoreParams(struct_size=8)
    assert be.lib.kllm_gpu_score_tokens(be.ctx, ctypes.byref(short)) == kb.EINVAL


@pytest.mark.parametrize("V", [128256, 33000])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_logits_of_zero_at_the_threshold(be, V, top):
    """A padding row of zeros has every logit at 0, and its alternatives are the
    lowest indices; so do rows with a few positive logits over many zeros."""
    R, K = 6, 64
    h, w = grid_case(R, K, V, V + top)
    h[:4] = 0
    w[:, :3] = 0
    h[1, 0] = h[2, 1] = h[3, 2] = 0.25
    w[::7, 0] = -0.125                       # zeros and below
    w[np.arange(0, V, V // 5), 1] = 0.125    # five or six above zero
    w[:, 2] = -0.125                         # nothing but the last few at zero
    w[V - 40:, 2] = 0
    got = check(be, h, w, some_targets(R, V, 2, 1), top)
    assert (got["top_ids"][0] == np.arange(top)).all()


@pytest.mark.parametrize("offset,temperature", [(0, None), (256, None), (0, 0.01), (256, 0.02),
                                                (-256, 0.02)])
def test_distances_to_the_maximum(be, offset, temperature):
    """Log-probabilities depend on the distance to the row's maximum alone: a
    common offset and a low temperature cost no accuracy, and none is above 0."""
    R, K, V = 70, 128, 9001
    h, w = grid_case(R, K, V, 31)
    h[:, 0], w[:, 0] = 16.0, offset / 16.0
    T = None if temperature is None else np.full(R, temperature)
    targets = some_targets(R, V, 3, 6)
    targets[:, 2] = (h @ w.T).argmax(1)
    got = run(be, h, w, targets, 20, T)
    want = sc.rows(h.astype(np.float64) @ w.astype(np.float64).T,
                   None if T is None else T.astype(np.float32), targets, 20)
    sc.assert_distances(got, want, V)


def test_the_likeliest_token_stays_at_or_below_zero(be):
    """A target's logit is a sum of its own order: it may round above the maximum
    of the tensor core's, and at a low temperature that would count."""
    rng = np.random.default_rng(15)
    R, K, V = 150, 2048, 3000
    h = wl.bf16_to_f32(wl.f32_to_bf16(rng.standard_normal((R, K)).astype(np.float32)))
    w = wl.bf16_to_f32(wl.f32_to_bf16((rng.standard_normal((V, K)) * 0.05).astype(np.float32)))
    logits = h.astype(np.float64) @ w.astype(np.float64).T
    best = logits.argmax(1)[:, None]
    got = run(be, h, w, best, 3, np.full(R, 1e-3))
    assert (got["logprob"] <= 0).all() and (got["top_logprobs"] <= 0).all()
    # a logit is off by K eps sum |h w|, each of the two in a distance
    err = 2 * K * sc.EPS * (np.abs(h).astype(np.float64) @ np.abs(w).T.astype(np.float64)).max(1)
    want = sc.rows(logits, np.full(R, 1e-3, np.float32), best, 3)
    sc.assert_near(got["logprob"], want["logprob"],
                   err[:, None] / 1e-3 + sc.distance_bound(want["entropy"], 0.0, V)[:, None], "best")


def test_contexts_in_threads_with_joins_of_different_sizes(be):
    """Two contexts on one GPU, each in a thread of its own: many ranges with 32
    alternatives (43 KB of the join's shared memory) and few without (a call's
    size must not become the other's limit)."""
    import threading

    import torch
    other = kb.Backend()
    cases = [(be, 128256, 32), (other, 200, 0)]
    rcs = [[], []]

    def calls(which):
        b, V, top = cases[which]
        h = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
        w = torch.zeros((V, 64), dtype=torch.bfloat16, device="cuda")
        f = torch.zeros((4, 32), device="cuda")
        i = torch.zeros((4, 32), dtype=torch.int32, device="cuda")
        nb = b.score_workspace_size(4, V, 0, top)
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for _ in range(400):
            rcs[which].append(b.score_tokens(
                hidden=h.data_ptr(), weight=w.data_ptr(), num_rows=4, hidden_dim=64, vocab=V,
                lse=f.data_ptr(), top_n=top, top_ids=i.data_ptr(), top_logprobs=f.data_ptr(),
                workspace=ws.data_ptr(), workspace_bytes=nb))
        torch.cuda.synchronize()

    threads = [threading.Thread(target=calls, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    other.close()
    assert rcs == [[0] * 400, [0] * 400]


def test_as_many_rows_as_a_call_takes(be):
    """2^20 rows: 512 groups of row blocks, offsets of the ranges' lists past 2^28
    bytes; checked on the GPU in 64 bits."""
    import torch
    R, K, V = 1 << 20, 64, 130
    gen = torch.Generator("cuda").manual_seed(3)
    h = (torch.randn((R, K), generator=gen, device="cuda") * 8).round().clamp(-32, 32) / 4
    w = (torch.randn((V, K), generator=gen, device="cuda") * 40).round().clamp(-127, 127) / 512
    h, w = h.bfloat16(), w.bfloat16()
    tgt = torch.randint(0, V, (R, 1), generator=gen, device="cuda", dtype=torch.int32)
    f = lambda *s: torch.full(s, 7.5, device="cuda")  # noqa: E731
    lp, lse, top = f(R, 1), f(R), f(R, 20)
    ids = torch.full((R, 20), -77, dtype=torch.int32, device="cuda")
    nb = be.score_workspace_size(R, V, 1, 20)
    ws = torch.full((nb + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert be.score_tokens(hidden=h.data_ptr(), weight=w.data_ptr(), num_rows=R, hidden_dim=K,
                           vocab=V, num_targets=1, targets=tgt.data_ptr(),
                           target_logprobs=lp.data_ptr(), lse=lse.data_ptr(), top_n=20,
                           top_ids=ids.data_ptr(), top_logprobs=top.data_ptr(),
                           workspace=ws.data_ptr(), workspace_bytes=nb, err_word=err.data_ptr(),
                           stream=torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert int(err.item()) == 0 and (ws[nb:] == 0xA5).all()
    for a in range(0, R, 1 << 17):
        b = a + (1 << 17)
        x = h[a:b].double() @ w.double().t()
        want = x.logsumexp(1)
        # |z| + ln V below 200: distance_bound and the rounding of lse at its size
        tol = sc.distance_bound(np.log(V), 200.0, V) + 4 * sc.EPS * 200.0
        assert ((lse[a:b].double() - want).abs() <= tol).all()
        assert ((lp[a:b].double() - (x.gather(1, tgt[a:b].long()) - want[:, None])).abs() <= tol).all()
        v, i = torch.sort(x, dim=1, descending=True, stable=True)
        assert torch.equal(ids[a:b].long(), i[:, :20])
        assert ((top[a:b].double() - (v[:, :20] - want[:, None])).abs() <= tol).all()

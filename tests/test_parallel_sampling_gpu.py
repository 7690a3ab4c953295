# SPDX-License-Identifier: Apache-2.0
"""examples/parallel_sampling.py end to end: layout, forks, prefill, append,
shared-prefix attention, lm_head and the scores together, each step's attention
and scores against 64 bits from the pages that the step could see."""
from __future__ import annotations

import importlib.util
import os

import numpy as np
import pytest

import scorecase as sc
import kllm_b200 as kb
from kllm_b200 import workloads as wl

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def ps():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "parallel_sampling.py")
    spec = importlib.util.spec_from_file_location("parallel_sampling", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


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


def cached(be, cache, rows, longest):
    """Every row's K and V as the pages hold them: [row][head][token][d] floats."""
    import torch
    m = cache.m
    n = cache.max_blocks * cache.block
    k = torch.zeros(rows, m.kv_heads, n, m.d, dtype=torch.int16, device="cuda")
    v = torch.zeros_like(k)
    cnt = torch.zeros(rows * m.kv_heads, dtype=torch.int32, device="cuda")
    rc = be.gather(k_out=k.data_ptr(), v_out=v.data_ptr(), counts_out=cnt.data_ptr(),
                   block_tables=cache.tables.data_ptr(), seq_lens=cache.lens.data_ptr(),
                   num_seqs=rows, num_kv_heads=m.kv_heads, head_dim=m.d,
                   max_blocks_per_seq=cache.max_blocks, block_size=cache.block,
                   kv_dtype=cache.kv, layer=0, layer_stride=2 * cache.page, stream=cache.stream)
    assert rc == 0
    torch.cuda.synchronize()
    return [wl.bf16_to_f32(x.cpu().numpy().view(np.uint16)).astype(np.float64)[:, :, :longest]
            for x in (k, v)]


@pytest.mark.parametrize("kv", [kb.KV_BF16, kb.KV_MX_FP8])
@pytest.mark.parametrize("lengths,samples,steps", [([160], 5, 4), ([77, 300, 16, 5], 9, 6)])
def test_samples_and_their_scores(be, ps, kv, lengths, samples, steps):
    import torch
    model = ps.Model(vocab=1000)
    rng = np.random.default_rng(len(lengths))
    prompts = [rng.integers(0, model.vocab, n).tolist() for n in lengths]
    trace = []
    r = ps.sample(be, model, prompts, samples, steps, top_n=7, kv=kv, trace=trace)
    P, R = len(prompts), len(prompts) * samples
    head = model.head.double()
    k, v = cached(be, r["cache"], P + R, max(lengths) + steps)
    f64 = lambda t: t.double().cpu().numpy()  # noqa: E731

    for i, step in enumerate(trace):
        if i > 0:
            q, got = f64(step["q"]), f64(step["attention"])
            scale = model.d ** -0.5
            for s in range(R):
                n = step["ctx"][s]
                for h in range(model.heads):
                    kk, vv = (x[P + s, h // (model.heads // model.kv_heads), :n] for x in (k, v))
                    x = kk @ q[s, h] * scale
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    e = 4 * model.d * EPS * (np.abs(kk) @ np.abs(q[s, h])).max() * scale
                    want = w @ vv
                    # as tests/prefixcase.py bounds it
                    tol = 1e-6 + 2.0 ** -8 * np.abs(want) + (2.0 ** -11 + 2 * e) * (w @ np.abs(vv))
                    assert (np.abs(got[s, h] - want) <= tol).all(), (i, s, h)
        logits = f64(step["logits"])
        exact = (step["hidden"].double() @ head.T).cpu().numpy()
        terms = (step["hidden"].double().abs() @ head.abs().T).cpu().numpy()
        assert (np.abs(logits - exact) <= 2 * model.hidden * EPS * terms).all()
        tokens = r["tokens"][i].cpu().numpy()
        want = sc.rows(logits, np.full(R, 0.8, np.float32), tokens[:, None], 7)
        lse_tol, ent_tol = sc.bounds(want, model.vocab)
        sc.assert_near(r["logprob"][i].cpu(), want["logprob"], lse_tol[:, None], "logprob")
        sc.assert_near(r["entropy"][i].cpu(), want["entropy"], ent_tol, "entropy")
        assert (r["rank"][i].cpu().numpy() == want["rank"]).all()
        assert (r["top_ids"][i].cpu().numpy() == want["top_ids"]).all()

    # the prompts' scores; a logit's fp32 sum is off by 2 K eps of its terms, a
    # log-probability by twice that, the entropy by as much times its weights
    for p, tokens in enumerate(prompts):
        hid = r["prompt_hidden"][p].double()
        targets = np.array([[t] for t in tokens[1:] + [-1]])
        want = sc.rows((hid @ head.T).cpu().numpy(), None, targets, 1)
        terms = (hid.abs() @ head.abs().T).amax(1).cpu().numpy() * 2 * 2 * model.hidden * EPS
        lse_tol, ent_tol = sc.bounds(want, model.vocab)
        sc.assert_near(r["prompt_logprob"][p].cpu()[:, None], want["logprob"],
                       (lse_tol + terms)[:, None], "prompt")
        sc.assert_near(r["prompt_entropy"][p].cpu(), want["entropy"],
                       ent_tol + terms * (4 + 2 * np.log(model.vocab)), "prompt entropy")


def test_forks_share_the_prompts_pages(be, ps):
    model = ps.Model(vocab=512)
    r = ps.sample(be, model, [list(range(70))], 3, 3, kv=kb.KV_BF16)
    t = r["cache"].tables.cpu().numpy().view(np.int64)
    assert (t[1:, :4] == t[0, :4]).all()                      # 64 of 70 tokens
    assert len({int(x) for x in t[:, 4, 0]}) == 4             # then a page each
    assert r["cache"].lens.tolist() == [70, 72, 72, 72]


def test_on_the_default_stream_and_on_a_side_stream(be, ps):
    """The calls run where torch's tensors are made: the same samples and scores
    whatever the current stream is."""
    import torch
    model = ps.Model(vocab=600)
    prompts = [list(range(100)), list(range(200, 230))]
    want = ps.sample(be, model, prompts, 4, 5, kv=kb.KV_BF16)
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            got = ps.sample(be, model, prompts, 4, 5, kv=kb.KV_BF16)
        for k in ("tokens", "logprob", "rank", "entropy", "top_ids"):
            assert torch.equal(got[k], want[k]), (k, stream)

# SPDX-License-Identifier: Apache-2.0
"""Several scored continuations of each prompt, on one GPU.

    python examples/parallel_sampling.py --prompts 2 --samples 16 --steps 24

A one-layer model with random weights stands in for a real one; what it shows
is the order of the calls and who owns what:

  prompts    kllm_gpu_batch_layout   pages and token rows of the prompts
             kllm_gpu_prefill_v2     attention over the prompts, their K/V cached
             kllm_gpu_score_tokens   log-probability of every prompt token, no
                                     logits stored
  forks      kllm_gpu_batch_layout   each sample's table starts with its prompt's
                                     whole pages; the tokens of the last, partial
                                     page go to a page of the sample's own
             kllm_gpu_kv_append_v2
  each step  kllm_gpu_batch_layout   a page for each sample that needs one
             kllm_gpu_kv_append_v2   the new tokens' K/V
             kllm_gpu_shared_prefix_attention
                                     the prompt's pages once for all its samples
             kllm_gpu_lm_head_sample logits and the next tokens
             kllm_gpu_logprobs       what each token's choice was worth, and the
                                     alternatives

The host only keeps lengths: it never waits for the GPU between the steps.
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "xpu-kllm_b200"))
import kllm_b200 as kb  # noqa: E402


class Model:
    """One attention layer between an embedding and an output matrix."""

    def __init__(self, vocab=4096, heads=4, kv_heads=2, seed=0):
        self.vocab, self.heads, self.kv_heads, self.d = vocab, heads, kv_heads, 128
        self.hidden = heads * self.d
        gen = torch.Generator("cuda").manual_seed(seed)

        def rand(rows, cols, std):
            x = torch.randn(rows, cols, generator=gen, device="cuda") * std
            return x.to(torch.bfloat16)

        self.embed = rand(vocab, self.hidden, 1.0)
        self.wq = rand(self.hidden, self.hidden, self.hidden ** -0.5)
        self.wk = rand(self.hidden, kv_heads * self.d, self.hidden ** -0.5)
        self.wv = rand(self.hidden, kv_heads * self.d, self.hidden ** -0.5)
        self.head = rand(vocab, self.hidden, 1.5 * self.hidden ** -0.5)

    def qkv(self, tokens):
        x = self.embed[tokens]
        return (x, (x @ self.wq).view(-1, self.heads, self.d),
                (x @ self.wk).view(-1, self.kv_heads, self.d),
                (x @ self.wv).view(-1, self.kv_heads, self.d))

    def out(self, x, attention):
        return x + attention.view(-1, self.hidden)


def _ok(rc):
    if rc != 0:
        raise RuntimeError(f"kllm_gpu call returned {rc}")


def _stream():
    """torch's current stream. Its default stream has the handle 0, which the
    library takes for its context's own stream; 1 names the default one."""
    return torch.cuda.current_stream().cuda_stream or 1


def _ptr(t):
    return t.data_ptr() if t is not None else None


class Cache:
    """The pages of S rows, their tables, and one layout call a step."""

    def __init__(self, be, model, rows, max_tokens, slots, block, kv):
        self.be, self.m, self.rows, self.block, self.kv = be, model, rows, block, kv
        self.max_blocks = -(-max_tokens // block)
        per_token = model.d * 9 // 8 if kv == kb.KV_MX_FP8 else model.d * 2
        self.page = model.kv_heads * block * per_token
        self.arena = torch.empty(slots, 2 * self.page, dtype=torch.uint8, device="cuda")
        i32 = dict(dtype=torch.int32, device="cuda")
        self.free = torch.randperm(slots, device="cuda").to(torch.int32)
        self.taken = 0
        self.tables = torch.zeros(rows, self.max_blocks, 24, dtype=torch.uint8, device="cuda")
        self.lens = torch.zeros(rows, **i32)
        self.cu = torch.zeros(rows + 1, **i32)
        self.err = torch.zeros(1, **i32)
        self.stream = _stream()

    def layout(self, ctx, new, forks=None):
        """Pages for `new` more tokens of each row; the token rows' sequence and
        position. Lengths are host lists, so the slots taken are known here."""
        i32 = dict(dtype=torch.int32, device="cuda")
        n = sum(new)
        seq, pos = torch.empty(max(n, 1), **i32), torch.empty(max(n, 1), **i32)
        c, w = torch.tensor(ctx, **i32), torch.tensor(new, **i32)
        f = torch.tensor(forks, **i32) if forks else None
        _ok(self.be.batch_layout(
            ctx_lens=_ptr(c), new_lens=_ptr(w), fork_from=_ptr(f),
            free_slots=self.free.data_ptr() + 4 * self.taken,
            num_free=self.free.numel() - self.taken, num_seqs=self.rows,
            max_blocks_per_seq=self.max_blocks, block_size=self.block,
            arena_base=self.arena.data_ptr(), slot_bytes=2 * self.page,
            total_slots=self.arena.shape[0], k_offset=0, v_offset=self.page,
            block_tables=_ptr(self.tables), seq_lens=_ptr(self.lens), cu_seqlens=_ptr(self.cu),
            token_seq=_ptr(seq), token_pos=_ptr(pos), token_capacity=max(n, 1),
            err_word=_ptr(self.err), stream=self.stream))
        self.taken += sum(-(-(a + b) // self.block) - -(-a // self.block) for a, b in zip(ctx, new))
        return seq, pos

    def paged(self, first_row=0):
        """Arguments that every call on the pages takes."""
        return dict(block_tables=self.tables[first_row].data_ptr(),
                    max_blocks_per_seq=self.max_blocks, num_kv_heads=self.m.kv_heads,
                    head_dim=self.m.d, block_size=self.block, kv_dtype=self.kv, layer=0,
                    layer_stride=2 * self.page, err_word=_ptr(self.err), stream=self.stream)

    def append(self, k, v, seq, pos):
        if k.shape[0]:
            _ok(self.be.append(k=_ptr(k), v=_ptr(v), token_seq=_ptr(seq), token_pos=_ptr(pos),
                               num_tokens=k.shape[0], num_seqs=self.rows, **self.paged()))


def sample(be, model, prompts, samples, steps, temperature=0.8, top_n=5, block=16,
           kv=kb.KV_MX_FP8, seed=0, trace=None):
    """`samples` continuations of `steps` tokens of each prompt (lists of token
    ids). Returns the prompts' log-probabilities, the tokens and their scores;
    with a list as `trace`, the queries and attentions of each step go there."""
    P, R, stream = len(prompts), len(prompts) * samples, _stream()
    length = [len(p) for p in prompts]
    whole = [n // block * block for n in length]
    slots = sum(-(-n // block) for n in length) + R * (-(-steps // block) + 2) + 8
    cache = Cache(be, model, P + R, max(length) + steps, slots, block, kv)
    gen = torch.Generator("cuda").manual_seed(seed)
    f32, i32 = dict(dtype=torch.float32, device="cuda"), dict(dtype=torch.int32, device="cuda")

    # ---- the prompts: pages, attention, scores -----------------------------------
    none = [0] * R
    cache.layout([0] * P + none, length + none)
    flat = torch.tensor([t for p in prompts for t in p], device="cuda")
    x, q, k, v = model.qkv(flat)
    attention = torch.empty_like(q)
    zero = torch.zeros(P, **i32)
    _ok(be.prefill(output=_ptr(attention), q=_ptr(q), k=_ptr(k), v=_ptr(v),
                   cu_seqlens=_ptr(cache.cu), ctx_lens=_ptr(zero), num_seqs=P,
                   num_tokens=len(flat), max_chunk=max(length), num_heads=model.heads,
                   scale=model.d ** -0.5, append=1, **cache.paged()))
    hidden = model.out(x, attention)
    nxt = torch.tensor([t for p in prompts for t in p[1:] + [-1]], **i32)   # -1: nothing follows
    scores = dict(logprob=torch.empty(len(flat), 1, **f32), entropy=torch.empty(len(flat), **f32))
    nb = be.score_workspace_size(len(flat), model.vocab, 1, 0)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    _ok(be.score_tokens(hidden=_ptr(hidden), weight=_ptr(model.head), num_rows=len(flat),
                        hidden_dim=model.hidden, vocab=model.vocab, num_targets=1,
                        targets=_ptr(nxt), target_logprobs=_ptr(scores["logprob"]),
                        entropy=_ptr(scores["entropy"]), workspace=_ptr(ws), workspace_bytes=nb,
                        err_word=_ptr(cache.err), stream=stream))

    # ---- the samples fork ------------------------------------------------------------
    of = [p for p in range(P) for _ in range(samples)]           # the prompt of each sample
    seq, pos = cache.layout(length + [whole[p] for p in of],
                            [0] * P + [length[p] - whole[p] for p in of], [-1] * P + of)
    first = [sum(length[:p]) for p in range(P)]
    tail = [first[p] + i for p in of for i in range(whole[p], length[p])]
    at = torch.tensor(tail, dtype=torch.long, device="cuda")
    cache.append(k[at].contiguous(), v[at].contiguous(), seq, pos)
    last = torch.tensor([first[p] + length[p] - 1 for p in of], device="cuda")
    prompt_hidden, hidden = hidden, hidden[last].contiguous()

    # ---- the steps ---------------------------------------------------------------------
    starts = torch.arange(0, R + 1, samples, **i32)
    shared = torch.tensor(whole, **i32)
    ctx = [length[p] for p in of]
    method = torch.full((R,), kb.SAMPLE_TEMPERATURE, **i32)
    temp = torch.full((R,), temperature, **f32)
    lws = torch.empty(be.lib.kllm_gpu_lm_head_workspace_size(min(R, 256), model.vocab),
                      dtype=torch.uint8, device="cuda")
    nb = be.shared_prefix_workspace_size(R, model.heads, model.kv_heads, model.d, cache.max_blocks)
    pws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    logits = torch.empty(R, model.vocab, **f32)
    out = dict(tokens=torch.empty(steps, R, **i32), logprob=torch.empty(steps, R, 1, **f32),
               rank=torch.empty(steps, R, 1, **i32), entropy=torch.empty(steps, R, **f32),
               top_ids=torch.empty(steps, R, top_n, **i32),
               top_logprob=torch.empty(steps, R, top_n, **f32))
    for i in range(steps):
        if i > 0:
            seq, pos = cache.layout(length + ctx, [0] * P + [1] * R)
            ctx = [c + 1 for c in ctx]
            x, q, k, v = model.qkv(out["tokens"][i - 1].long())
            cache.append(k, v, seq, pos)
            attention = torch.empty_like(q)
            _ok(be.shared_prefix(output=_ptr(attention), query=_ptr(q),
                                 seq_lens=cache.lens[P:].data_ptr(), group_starts=_ptr(starts),
                                 prefix_lens=_ptr(shared), num_seqs=R, num_groups=P,
                                 num_heads=model.heads, scale=model.d ** -0.5,
                                 workspace=_ptr(pws), workspace_bytes=nb, **cache.paged(P)))
            hidden = model.out(x, attention)
        draw = torch.rand(R, generator=gen, **f32)
        for a in range(0, R, 256):                       # the projection takes 256 rows
            b = min(R, a + 256)
            _ok(be.lm_head(hidden=_ptr(hidden[a:b]), weight=_ptr(model.head), num_rows=b - a,
                           hidden_dim=model.hidden, vocab=model.vocab, logits=_ptr(logits[a:b]),
                           method=_ptr(method[a:b]), temperature=_ptr(temp[a:b]),
                           uniform=_ptr(draw[a:b]), tokens=_ptr(out["tokens"][i, a:b]),
                           workspace=_ptr(lws), workspace_bytes=lws.numel(),
                           err_word=_ptr(cache.err), stream=stream))
        _ok(be.logprobs(logits=_ptr(logits), logits_dtype=0, num_rows=R, vocab=model.vocab,
                        num_targets=1, temperature=_ptr(temp), targets=_ptr(out["tokens"][i]),
                        target_logprobs=_ptr(out["logprob"][i]), target_ranks=_ptr(out["rank"][i]),
                        entropy=_ptr(out["entropy"][i]), top_n=top_n,
                        top_ids=_ptr(out["top_ids"][i]), top_logprobs=_ptr(out["top_logprob"][i]),
                        stream=stream))
        if trace is not None:
            trace.append(dict(q=q, attention=attention, hidden=hidden, logits=logits.clone(),
                              ctx=list(ctx)))
    torch.cuda.synchronize()
    if int(cache.err):
        raise RuntimeError(f"error word 0x{int(cache.err):x}")
    return dict(out, prompt_logprob=scores["logprob"][:, 0].split(length),
                prompt_entropy=scores["entropy"].split(length),
                prompt_hidden=prompt_hidden.split(length), cache=cache)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", type=int, default=2)
    ap.add_argument("--length", type=int, default=500)
    ap.add_argument("--samples", type=int, default=16)
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--kv", choices=["mx", "bf16"], default="mx")
    a = ap.parse_args()
    be = kb.Backend()
    if be.backend != kb.KLLM_GPU_CUDA:
        raise SystemExit("no sm_100 device")
    with torch.cuda.stream(be.torch_stream()):
        model = Model()
        rng = torch.Generator().manual_seed(1)
        prompts = [torch.randint(0, model.vocab, (a.length + 7 * p,), generator=rng).tolist()
                   for p in range(a.prompts)]
        r = sample(be, model, prompts, a.samples, a.steps, a.temperature,
                   kv=kb.KV_MX_FP8 if a.kv == "mx" else kb.KV_BF16)
    for p in range(a.prompts):
        mean = r["prompt_logprob"][p][:-1].mean().item()
        print(f"prompt {p}: {len(prompts[p])} tokens, perplexity {math.exp(-mean):.1f}")
        rows = slice(p * a.samples, (p + 1) * a.samples)
        total = r["logprob"][:, rows, 0].sum(0)
        for s in total.argsort(descending=True)[:3].tolist():
            tok = r["tokens"][:, p * a.samples + s].tolist()
            print(f"  sample {s:3d}: log-probability {total[s]:8.2f}  tokens {tok[:8]} ...")
    be.close()


if __name__ == "__main__":
    main()

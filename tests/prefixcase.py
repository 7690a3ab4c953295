# SPDX-License-Identifier: Apache-2.0
"""Paged caches whose sequences share their leading pages, for the parity
tests of kllm_gpu_shared_prefix_attention: one arena, block tables for host
and device, and the attention of each row in 64 bits."""
from __future__ import annotations

import numpy as np

import kvcase
import oracle
from kllm_b200 import workloads as wl

EPS = 2.0 ** -24


class PrefixCase:
    """groups: list of (prefix tokens, [context length of each row]). Rows that
    hold the prefix share its whole pages; every other page is a row's own.
    loose: context lengths of rows after the last group (in no group)."""

    def __init__(self, cfg, groups, seed=0, loose=(), max_blocks=None, magnitude=2.0):
        rng = np.random.default_rng(seed)
        self.cfg, bs = cfg, cfg.block
        self.starts = np.concatenate([[0], np.cumsum([len(r) for _, r in groups])]).astype(np.int32)
        self.plens = np.array([p for p, _ in groups], np.int32)
        self.lens = np.array([n for _, r in groups for n in r] + list(loose), np.int32)
        S = len(self.lens)
        nblk = -(-np.maximum(self.lens, 0) // bs)
        self.max_blocks = int(max_blocks or max(1, nblk.max()))
        slots = np.full((S, self.max_blocks), -1, np.int64)
        used = 0
        for g, (p, rows) in enumerate(groups):
            k = max(0, int(p)) // bs
            for i, n in enumerate(rows):
                s = self.starts[g] + i
                if n >= k * bs:
                    slots[s, :k] = np.arange(used, used + k)
            used += k
        for s in range(S):
            own = np.flatnonzero((slots[s] < 0) & (np.arange(self.max_blocks) < nblk[s]))
            slots[s, own] = np.arange(used, used + len(own))
            used += len(own)
        perm = rng.permutation(used + 3)
        self.slots = np.where(slots >= 0, perm[slots], -1)
        self.valid = self.slots >= 0
        self.arena = np.zeros((used + 3, cfg.layers, 2, cfg.page_bytes()), np.uint8)
        for layer in range(cfg.layers):
            for which in range(2):
                x = wl.f32_to_bf16((rng.standard_normal(((used + 3) * bs, cfg.hkv, cfg.d)) *
                                    magnitude).astype(np.float32))
                pay, sc = oracle.mx_quantize(x) if cfg.kv_dtype == wl.KV_MX_FP8 else (x, None)
                self.arena[:, layer, which] = kvcase._pages_from_rows(cfg, pay, sc, used + 3, 0)
        self.q = wl.f32_to_bf16(rng.standard_normal((S, cfg.hq, cfg.d)).astype(np.float32))

    def table(self, base):
        t = np.zeros(self.slots.shape, wl.ENTRY_DTYPE)
        a = base + self.slots * self.cfg.slot_bytes()
        t["k"] = np.where(self.valid, a, 0)
        t["v"] = np.where(self.valid, a + self.cfg.page_bytes(), 0)
        t["valid"] = self.valid
        return t

    def want(self, layer=0):
        """(output, bound) in 64 bits: the attention of each row over the tokens
        of its own table. The bound: bf16 output (2^-8 of it, half for the
        rounding), P to 11 bits (2^-11 of sum p |v|, twice its rounding), scores
        as fp32 sums of d products (an error e of a score weighs p by e)."""
        c = self.cfg
        table = np.ascontiguousarray(self.table(self.arena.ctypes.data))
        off = layer * c.layer_stride()
        out = np.zeros((len(self.lens), c.hq, c.d))
        tol = np.full_like(out, 1e-6)
        q = wl.bf16_to_f32(self.q).astype(np.float64)
        for s, n in enumerate(self.lens):
            for h in range(c.hkv):
                k, v = oracle.gather(table[s], self.max_blocks, int(max(n, 0)), h, c.hkv, c.d,
                                     c.block, c.kv_dtype, off)
                if len(k) == 0:
                    continue
                k, v = (wl.bf16_to_f32(x).astype(np.float64) for x in (k, v))
                for i in range(h * c.group, (h + 1) * c.group):
                    x = k @ q[s, i] * c.scale
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    e = 4 * c.d * EPS * (np.abs(k) @ np.abs(q[s, i])).max() * c.scale
                    out[s, i] = w @ v
                    tol[s, i] += 2.0 ** -8 * np.abs(out[s, i]) + (2.0 ** -11 + 2 * e) * (w @ np.abs(v))
        return out, tol


class OnDevice:
    def __init__(self, case):
        import torch
        self.case = case
        self.arena = torch.from_numpy(case.arena).cuda()
        self.set_table()
        up = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
        self.lens, self.starts, self.plens = up(case.lens), up(case.starts), up(case.plens)
        self.q = torch.from_numpy(case.q.view(np.int16)).cuda()
        S, c = len(case.lens), case.cfg
        self.out = torch.full((S, c.hq, c.d), 0x7FC0, dtype=torch.int16, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def set_table(self):
        import torch
        t = self.case.table(self.arena.data_ptr())
        self.tab = torch.from_numpy(t.view(np.uint8).copy()).cuda()

    def kwargs(self, **over):
        c, d = self.case.cfg, self.case
        kw = dict(output=self.out.data_ptr(), query=self.q.data_ptr(),
                  block_tables=self.tab.data_ptr(), seq_lens=self.lens.data_ptr(),
                  group_starts=self.starts.data_ptr(), prefix_lens=self.plens.data_ptr(),
                  num_seqs=len(d.lens), num_groups=len(d.plens), num_heads=c.hq,
                  num_kv_heads=c.hkv, head_dim=c.d, max_blocks_per_seq=d.max_blocks,
                  block_size=c.block, kv_dtype=c.kv_dtype, layer=0, scale=c.scale,
                  layer_stride=c.layer_stride(), err_word=self.err.data_ptr())
        kw.update(over)
        return kw

    def run(self, be, **over):
        """The call with a workspace of rubbish; returns the outputs as float."""
        import torch
        c, d = self.case.cfg, self.case
        self.out.fill_(0x7FC0)
        self.err.zero_()
        nb = be.shared_prefix_workspace_size(len(d.lens), c.hq, c.hkv, c.d, d.max_blocks)
        assert nb > 0
        ws = torch.full((nb + 256,), 0xA5, dtype=torch.uint8, device="cuda")
        kw = self.kwargs(workspace=ws.data_ptr(), workspace_bytes=nb,
                         stream=torch.cuda.current_stream().cuda_stream)
        kw.update(over)
        rc = be.shared_prefix(**kw)
        assert rc == 0, (rc, be.stats().last_cuda_error)
        torch.cuda.synchronize()
        assert (ws[nb:] == 0xA5).all(), "written past the workspace"
        return wl.bf16_to_f32(self.out.cpu().numpy().view(np.uint16))


def assert_near(got, want, what=""):
    out, tol = want
    assert np.isfinite(got).all(), f"{what}: non-finite output"
    r = np.abs(got - out) / tol
    assert r.max() <= 1.0, (what, float(r.max()), np.unravel_index(r.argmax(), r.shape))

# SPDX-License-Identifier: Apache-2.0
"""Definitions in 64 bits of the scoring operators (log-probabilities, ranks,
entropy, top alternatives) and of the batch layout, written row by row, and
the error bounds their 32-bit kernels are held to."""
from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24        # half a unit in the last place of fp32


def rows(logits, temperature, targets, top_n):
    """logits float64 [R, V] -> dict of arrays; the rules of kllm_gpu_logprobs."""
    logits = np.asarray(logits, np.float64)
    R, V = logits.shape
    nt = targets.shape[1]
    out = dict(lse=np.zeros(R), entropy=np.zeros(R), logprob=np.zeros((R, nt)),
               rank=np.zeros((R, nt), np.int64), top_ids=np.zeros((R, top_n), np.int64),
               top_logprobs=np.zeros((R, top_n)), zmax=np.zeros(R))
    for r in range(R):
        l = logits[r]
        T = 1.0 if temperature is None or not temperature[r] > 0 else float(temperature[r])
        z = l / T
        fin = z[np.isfinite(z)]
        out["zmax"][r] = np.abs(fin).max() if fin.size else 0.0
        if np.isnan(l).any() or (l == np.inf).any():
            lse = ent = floor = np.nan
        elif (l == -np.inf).all():
            lse, ent, floor = -np.inf, 0.0, 0.0
        else:
            m = z.max()
            e = np.exp(z - m)
            s = e.sum()
            lse = floor = m + np.log(s)
            with np.errstate(invalid="ignore"):
                ent = np.log(s) - np.where(e > 0, e * (z - m), 0.0).sum() / s
        out["lse"][r], out["entropy"][r] = lse, ent
        for j, t in enumerate(targets[r]):
            if not 0 <= t < V:
                out["logprob"][r, j], out["rank"][r, j] = -np.inf, -1
                continue
            out["logprob"][r, j] = z[t] - floor
            with np.errstate(invalid="ignore"):
                out["rank"][r, j] = -1 if np.isnan(l[t]) else int(
                    (l > l[t]).sum() + (l[:t] == l[t]).sum())
        v = np.where(np.isnan(l), -np.inf, l)
        order = np.argsort(-v, kind="stable")[:top_n]
        out["top_ids"][r] = order
        out["top_logprobs"][r] = v[order] / T - floor
    return out


def bounds(want, V):
    """Absolute error bounds of the fp32 kernels, per row: (lse and logprobs,
    entropy). y = l c is off by 4 eps |y| (two constants, one product, one
    fma), each 2^(y - m) by that much times ln 2 and the exponential's 2^-22;
    a thread adds at most V / 512 + 64 terms and the joins 32 more; the last
    subtraction and products round |z| + |lse| a few times. The entropy's
    second sum weighs the same errors with |y - m|, on average at most the
    entropy itself + 2 in natural units."""
    z = want["zmax"]
    rel = 8 * EPS * z + 2.0 ** -22 + (V / 512 + 96) * EPS
    lse = rel + 8 * EPS * (z + np.log(V) + 1)
    return lse, (rel + 8 * EPS) * (4 + 2 * np.log(V))


def assert_near(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tol = np.broadcast_to(np.asarray(tol), want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = np.isfinite(want)
    assert (np.isnan(got) == np.isnan(want)).all(), f"{what}: NaNs differ"
    inf = ~fin & ~np.isnan(want)
    assert (got[inf] == want[inf]).all(), f"{what}: infinities differ"
    err = np.abs(got[fin] - want[fin])
    assert np.isfinite(err).all() and (err <= tol[fin]).all(), (
        what, float((err / tol[fin]).max()), got[fin][np.argmax(err / tol[fin])])


def distance_bound(entropy, distance, V):
    """Absolute bound of a log-probability that is formed from its distance D to
    the row's maximum and the logarithm of the sum S relative to it. The distance
    is one subtraction, one division and one product (3 eps D) and enters one
    more; ln S takes four roundings of at most ln V. A term of S is 2^d with d off
    by 5 eps of itself (D times two constants, on average the entropy at most) and
    the exponential's 2^-22; each raise of a thread's maximum (one a batch of at
    least 4,096 elements a CTA) and each of up to 16 joins is such a factor too,
    and a thread adds at most V / 512 + 64 terms, the joins 32 more."""
    rel = 5 * EPS * entropy + (V / 4096 + 17) * 2.0 ** -22 + (V / 512 + 96) * EPS
    return rel + 4 * EPS * distance + 5 * EPS * (np.log(V) + 1)


def assert_distances(got, want, V):
    """Log-probabilities within distance_bound, whatever the logits' size, and
    none above 0; the entropy weighs each term's error by its distance, on average
    the entropy itself; lse alone keeps the size of the logits."""
    ent = want["entropy"]
    for k in ("logprob", "top_logprobs"):
        dist = np.maximum(0.0, want["top_logprobs"][:, :1] - want[k])
        assert (got[k] <= 0).all(), k
        assert_near(got[k], want[k], distance_bound(ent[:, None], dist, V), k)
    tol = distance_bound(ent, 0.0, V)
    assert_near(got["entropy"], want["entropy"], 2 * tol * (1 + ent) + tol, "entropy")
    assert (got["entropy"] >= 0).all()
    assert_near(got["lse"], want["lse"], tol + 4 * EPS * want["zmax"], "lse")
    assert (got["top_ids"] == want["top_ids"]).all()


def layout(ctx_lens, new_lens, fork_from, free, table, *, block, base, slot_bytes, total, k_off,
           v_off, capacity):
    """Batch layout by its rules, one row and one token at a time. table:
    int64 [S, max_blocks, 3], changed in place."""
    S, mb, _ = table.shape
    cap = mb * block
    err, at = 0, 0
    seq_lens, cu = [], [0]
    token_seq = np.full(capacity, -1, np.int32)
    token_pos = np.zeros(capacity, np.int32)
    slot_map = np.full(capacity, -1, np.int64)
    old_table = table.copy()
    for s in range(S):
        c, n = max(int(ctx_lens[s]), 0), max(int(new_lens[s]), 0)
        if c > cap or n > cap - min(c, cap):
            err |= 0x1
        c = min(c, cap)
        n = min(n, cap - c)
        p = -1 if fork_from is None else int(fork_from[s])
        if p >= 0:
            if not (p < S and p != s and c % block == 0 and fork_from[p] < 0
                    and c <= min(max(int(ctx_lens[p]), 0), cap)):
                c = n = 0
                err |= 0x80
            else:
                table[s, :c // block] = old_table[p, :c // block]
        for j in range(-(-c // block), -(-(c + n) // block)):
            slot = int(free[at]) if at < len(free) else -1
            at += 1
            if 0 <= slot < total:
                a = base + slot * slot_bytes
                table[s, j] = (a + k_off, a + v_off, 1)
            else:
                table[s, j] = 0
                err |= 0x80
        for i in range(n):
            t, pos = cu[-1] + i, c + i
            if t >= capacity:
                err |= 0x80
                continue
            e = table[s, pos // block]
            token_seq[t], token_pos[t] = s, pos
            if int(e[2]) & 0xffffffff:
                slot_map[t] = (int(e[0]) - base - k_off) // slot_bytes * block + pos % block
        seq_lens.append(c + n)
        cu.append(cu[-1] + n)
    return dict(table=table, seq_lens=np.array(seq_lens, np.int32), cu=np.array(cu, np.int32),
                token_seq=token_seq, token_pos=token_pos, slot_map=slot_map,
                counts=np.array([cu[-1], at], np.int32), err=err)

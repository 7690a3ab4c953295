# SPDX-License-Identifier: Apache-2.0
"""The scoring operators without a GPU: struct layouts against the C header,
refusals before a device is touched, and the 64-bit definitions themselves."""
from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest

import scorecase as sc
import kllm_b200 as kb

STRUCTS = {
    "kllm_gpu_batch_layout_params": kb.BatchLayoutParams,
    "kllm_gpu_logprobs_params": kb.LogprobsParams,
    "kllm_gpu_score_params": kb.ScoreParams,
    "kllm_gpu_shared_prefix_params": kb.SharedPrefixParams,
}


def test_struct_layouts_match_c(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "kllm_gpu.h"',
             "int main(void) {"]
    for cname, cls in STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof(struct {cname}));')
        for f, _ in cls._fields_:
            lines.append(f'printf("{cname}.{f} %zu\\n", offsetof(struct {cname}, {f}));')
    lines.append('printf("limits %d %d %d\\n", KLLM_MAX_TOP_N, KLLM_MAX_TARGETS, KLLM_ERR_LAYOUT);')
    lines.append("return 0; }")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.dirname(kb.HEADER_PATH),
                    str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    got = {ln.split()[0]: ln.split()[1:] for ln in out.splitlines()}
    for cname, cls in STRUCTS.items():
        assert int(got[cname][0]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"][0]) == getattr(cls, f).offset, f"{cname}.{f}"
    assert [int(x) for x in got["limits"]] == [kb.MAX_TOP_N, kb.MAX_TARGETS, kb.ERR_LAYOUT]


def _gpu_present() -> bool:
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


@pytest.mark.skipif(_gpu_present(), reason="checks the no-device behaviour")
def test_no_device_is_refused():
    be = kb.Backend()
    assert be.batch_layout() == kb.ENODEV
    assert be.logprobs() == kb.ENODEV
    assert be.score_tokens() == kb.ENODEV
    assert be.shared_prefix() == kb.ENODEV and be.shared_prefix(flags=1) == kb.EINVAL
    assert be.shared_prefix_workspace_size(2, 32, 8, 128, 4) == 0
    assert be.score_workspace_size(4, 1000, 1, 5) == 0
    assert be.batch_layout(flags=1) == kb.EINVAL
    assert be.logprobs(flags=1) == kb.EINVAL
    assert be.score_tokens(flags=1) == kb.EINVAL
    be.close()


def test_definition_of_the_scores():
    p = np.array([0.5, 0.25, 0.125, 0.125])
    got = sc.rows(np.log(p)[None], None, np.array([[1, 2, 3, 4]]), 4)
    assert np.allclose(got["entropy"], -(p * np.log(p)).sum())
    assert np.allclose(got["logprob"][0, :3], np.log(p[1:]))
    assert got["rank"][0].tolist() == [1, 2, 3, -1] and np.isneginf(got["logprob"][0, 3])
    assert got["top_ids"][0].tolist() == [0, 1, 2, 3]
    assert abs(float(got["lse"][0])) < 1e-12
    dead = sc.rows(np.full((1, 3), -np.inf), None, np.array([[2]]), 2)
    assert np.isneginf(dead["lse"]).all() and dead["entropy"][0] == 0
    assert dead["rank"][0, 0] == 2 and dead["top_ids"][0].tolist() == [0, 1]


def test_definition_of_the_layout():
    table = np.zeros((3, 4, 3), np.int64)
    table[0, 0] = (1000, 1500, 1)          # slot 1 holds row 0's first block
    got = sc.layout([16, 3, 16], [2, 0, 1], [-1, -1, 0], np.array([5, 6, 7, 8]), table, block=16,
                    base=0, slot_bytes=1000, total=100, k_off=0, v_off=500, capacity=5)
    assert got["cu"].tolist() == [0, 2, 2, 3] and got["seq_lens"].tolist() == [18, 3, 17]
    assert got["token_seq"].tolist() == [0, 0, 2, -1, -1]
    assert got["token_pos"].tolist() == [16, 17, 16, 0, 0]
    assert got["slot_map"].tolist() == [80, 81, 96, -1, -1]
    assert got["table"][2, 0].tolist() == [1000, 1500, 1]     # the parent's block
    assert got["counts"].tolist() == [3, 2] and got["err"] == 0


def test_the_joins_shared_memory_is_no_function_attribute():
    """An attribute is the function's for every context and thread of a device: a
    size that changes from call to call would limit another thread's launch."""
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(kb.__file__))), "csrc",
                       "score.cu")
    with open(src) as f:
        text = f.read()
    calls = text.split("cudaFuncSetAttribute(")[1:]
    assert len(calls) == 1 and calls[0].startswith("score_kernel,")
    assert "static_assert(join_smem(kMaxSplits, KLLM_MAX_TOP_N_I) + 1024 <= 48 * 1024" in text

# SPDX-License-Identifier: Apache-2.0
"""Register hand-overs between warps, read from the CUDA sources. All four warps
of a warpgroup have to execute the same setmaxnreg, or the launch's registers
are not handed over; so the only ones stand in split_registers, whose compile
time checks hold the split to whole warpgroups and to the launch's registers."""
from __future__ import annotations

import os
import re

import kllm_b200 as kb

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(kb.__file__))), "csrc")


def sources():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh")):
            with open(os.path.join(CSRC, name)) as f:
                yield name, f.read()


def body(text, head):
    """The braces' content that follows `head`."""
    at = text.index("{", text.index(head))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError(head)


def test_every_setmaxnreg_stands_before_the_roles():
    found = 0
    for name, text in sources():
        n = len(re.findall(r'"setmaxnreg\.', text))
        if n == 0:
            continue
        helper = body(text, "bool split_registers(int warp)")
        assert len(re.findall(r'"setmaxnreg\.', helper)) == n == 2, name
        assert "FIRST % 4 == 0 && rest % 4 == 0" in helper
        found += 1
    assert found == 1


def test_the_roles_of_a_warpgroup_share_their_split():
    text = dict(sources())["shared_prefix.cu"]
    const = {k: int(v) for k, v in re.findall(r"(kWarp\w+) = (\d+)", text)}
    calls = re.findall(r"split_registers<(\w+), (\d+), (\d+)>\(warp\)", text)
    assert len(calls) == 2
    for first, hi, lo in calls:
        # SW<0>::N, the BF16 suffix CTA's working warps, is 8
        n = const.get(first, 8)
        assert n % 4 == 0 and n * int(hi) + (16 - n) * int(lo) <= 16 * 128

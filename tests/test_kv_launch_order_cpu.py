"""The cache's kernels start while their predecessor on the stream still runs:
in their source, each waits for it (or, where that one wrote none of them and
waited itself, fences) before it reads its inputs, and none reads them by loads
that ask for memory which stays unwritten."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "test_speed_scalesweep_b200", "csrc")
FILES = ("kv_write.cu", "kv_attend.cu", "kv_prompt.cu", "kv_pages.cu")


def source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def kernels():
    for name in FILES:
        text = source(name)
        for m in re.finditer(r"__global__", text):
            at = text.index("{", m.end())
            depth, end = 1, at + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            yield re.search(r"(\w+)\s*\(const", text[m.end():at]).group(1), text[at + 1:end - 1]


@pytest.mark.parametrize("name", FILES + ("attend.cuh",))
def test_no_non_coherent_loads(name):
    assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", source(name))


def test_every_kernel_waits_before_it_reads():
    found = dict(kernels())
    assert {"write_kernel", "gather_kernel", "decode_kernel", "join_kernel", "prompt_kernel", "prompt_wide_kernel",
            "fork_plan", "extend_slots", "compact_apply", "copy_kernel", "free_kernel"} <= set(found)
    # what reads the tables, the inputs or the workspace
    reads = re.compile(r"tile_of\(|decode_tile|rotate_query_unit|quantize_units|cache\.multiplier|slots\b.*\[|"
                       r"a\.seqs\[|a\.other\[|a\.refcount|a\.seq_lens|block_table|w\.head|copy_pairs")
    for name, body in found.items():
        wait = body.index("wait_for_predecessor()")
        ordered = min(wait, body.index("__threadfence()")) if name in ("join_kernel", "decode_kernel") else wait
        first = reads.search(body)
        assert first and ordered < first.start(), name
        assert body.index("let_successor_start()") > wait, name
    join = found["join_kernel"]  # the other grid's results only behind the wait
    assert join.rindex("wait_for_predecessor()") < join.index("ml[")

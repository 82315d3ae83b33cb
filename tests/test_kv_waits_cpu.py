"""Attention's bounded waits, in the source: every one says that it gave up, and
what it leaves unfinished becomes NaN, whether or not the caller passed a
status (the model of tests/test_kv_protocol_cpu.py says why that is enough)."""
import re

from test_kv_launch_order_cpu import kernels, source


def test_every_wait_of_the_prompt_kernels_marks_its_rows():
    found = dict(kernels())
    for name in ("prompt_kernel", "prompt_wide_kernel"):
        body = found[name]
        head, tail = body.split("auto wait = ", 1)
        assert "warp_wait" not in head and "mbar_wait" not in body
        assert tail.count("warp_wait(") == 1 and "give_up(ctl);" in tail[:300]
        # set before the warp goes on, looked at before the rows are stored, drained before TMEM goes
        mark, store = body.index("if (!ok || gave_up(ctl)) l = NAN;"), body.index("store_result<kD>(")
        assert mark < store < body.index("drain_after_giving_up(ctl)") < body.index("tcgen05.dealloc")
        assert "if (!ok && a.status && lane == 0) atomicCAS(a.status, 0, 1);" in body
        assert body.index("ctl->gave_up = 0;") < body.index("__syncthreads()")


def test_a_decode_warp_that_gave_up_leaves_nan():
    text = source("kv_attend.cu")
    assert "mbar_wait(" not in text.replace("warp_wait", "")
    at = text.index("if (!ok) {")
    assert re.search(r"l\[n\]\[0\] = l\[n\]\[1\] = NAN;", text[at:at + 300]) and at < text.index("float* mine")

"""CPU check of how device error words reach the host: every translation unit with a bounded wait
owns a word, and each word is read by obn_check_device_errors. No wait is made to run out on a GPU:
the words' way is followed in the sources."""
import os
import re

import pytest

from _util import ROOT

CSRC = os.path.join(ROOT, "0xbitnet_b200", "csrc")
WAITS = re.compile(r"\b(record_error|mbar_wait\w*|wait_or_abort\w*|q8_wait|mma_wait)\s*\(")


def text(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def included(name, seen=None):
    """name and every header of this folder that it includes, directly or not."""
    seen = set() if seen is None else seen
    if name not in seen and os.path.exists(os.path.join(CSRC, name)):
        seen.add(name)
        for h in re.findall(r'#include "([^"/]+)"', text(name)):
            included(h, seen)
    return seen


UNITS = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu") and WAITS.search(text(f)))


def test_the_units_with_waits():
    assert {"attention.cu", "gemm.cu", "gemv_mma.cu", "kernels.cu", "kvq8_attn.cu", "kvq8_many.cu",
            "lmhead.cu", "logits.cu"} <= set(UNITS)


@pytest.mark.parametrize("unit", UNITS)
def test_unit_lists_its_error_word(unit):
    """The word, its reader and the reader's listing stand in one header, with internal linkage,
    so that a unit which can record an error cannot be without them."""
    assert "obn_common.cuh" in included(unit)
    assert not re.search(r"__device__\s+uint32_t\s+g_dev_error", text(unit))
    common = text("obn_common.cuh")
    assert re.search(r"static __device__ uint32_t g_dev_error\b", common)
    reader = re.search(r"static cudaError_t (\w+)\(uint32_t\* out\) \{(.*?)\n\}", common, re.S)
    assert "cudaMemcpyFromSymbol(out, g_dev_error" in reader[2]
    assert "cudaMemcpyToSymbol(g_dev_error" in reader[2]
    assert re.search(r"static const bool \w+\s*=\s*list_dev_error\(&" + reader[1] + r"\);", common)


def test_the_check_reads_every_listed_word():
    body = re.search(r"cudaError_t read_and_clear_dev_error\(uint32_t\* out\) \{(.*?)\n\}",
                     text("kernels.cu"), re.S)[1]
    assert re.search(r"for \(DevErrorReader (\w+) : dev_error_readers\(\)\)", body)
    assert "read_and_clear_dev_error(&word)" in text("abi.cu")


def test_an_aborted_share_of_many_rows_leaves_nan():
    """After the softmax loop, which a wait that gives up leaves before the share is done, each
    warp fills the rows that are its own to write, to the end of the share."""
    src = text("kvq8_many.cu")
    after = src[src.index("for (int u = 0; cur.left > 0; ++u)"):src.index("} else if (warp < 20)")]
    fill = re.search(r"\n    \}\s*while \(cur\.left > 0\) \{(.*)", after, re.S)[1]
    assert "q8_next(sc, nxt)" in fill and "cur = nxt;" in fill
    assert re.search(r"i < row0 \+ 16;", fill) and "make_float4(nan, nan, nan, nan)" in fill
    assert "q8_part_o(ws, kRows, slot)" in fill and "out +" in fill


def test_a_late_copy_of_logits_leaves_nan_and_no_token():
    """The block agrees on a copy that did not come, uses nothing of it, waits for what is in
    flight, fills the rest with NaN and lets no other block's maximum win."""
    src = text("logits.cu")
    assert re.search(r"dead = __syncthreads_or\(wait && !mbar_wait\(&sm\.full\[buf\][^;]*;\s*"
                     r"if \(dead\) break;", src)
    late = src[src.index("if (dead) {"):src.index("if (!token) return;")]
    assert late.count("mbar_wait(&sm.full[") == 2
    assert re.search(r"y_row\[p - mis\] = __int_as_float\(0x7FC00000\);", late)
    assert "mine = dead ? 0xFFFFFFFFu" in src

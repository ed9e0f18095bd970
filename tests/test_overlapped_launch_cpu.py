"""Kernels launched before the one ahead of them has ended: none reads or writes memory before it
waits for the stream (shown by reading the sources; a stale read need not show on a GPU)."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tiledattention_b200", "csrc")


def _kernels():
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith(".cu"):
            continue
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        if "launch_overlapped" not in text:
            continue
        for m in re.finditer(r"__global__[^{;]*?(\w+)\((?:[^()]|\([^()]*\))*\)\s*\{", text):
            end = text.find("\n}", m.end())
            yield name, m.group(1), text[m.end():end]


def test_kernels_wait_before_they_touch_memory():
    found = list(_kernels())
    assert {k for _, k, _ in found} >= {"append_kernel", "attend_kernel", "merge_kernel", "chunk_kernel",
                                        "rotary_vector_kernel", "rotary_scalar_kernel"}
    for file, kernel, body in found:
        before, waits, _ = body.partition("wait_for_stream();")
        assert waits, (file, kernel)
        # p holds sizes and pointers: an indexed or dereferenced member, or a helper that does it
        for touch in (r"\bp\.\w+\[", r"\*p\.", r"extent_of\(", r"place_of\(", r"head_at\(", r"position_of\(",
                      r"checked_page\(", r"atomic\w+\(", r"reinterpret_cast<const (?:float|u?int)[24]\*>", r"__ldg",
                      r"tma_load", r"let_next_kernel_in"):
            assert not re.search(touch, before), (file, kernel, touch)
        assert not re.search(r"\breturn\b", before), (file, kernel)

"""The kernels of a CUDA source as text, without comments: what has to stand in which order, and what may not stand at all."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tandemllm_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", " ", f.read(), flags=re.S)


def _closed(text, at, pair):
    """The place behind the bracket that closes the one at `at`."""
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == pair[0]) - (text[i] == pair[1])
        if depth == 0:
            return i + 1
    raise ValueError("a bracket is not closed")


def kernels(name):
    """{kernel: (its parameters, its body)} of a source in csrc/."""
    text, out = source(name), {}
    for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\s*)?", text):
        at = m.end()
        if text[at] == "(":
            at = _closed(text, at, "()")
        called = re.compile(r"\s*(\w+)\s*\(").match(text, at)
        end = _closed(text, called.end() - 1, "()")
        body = text.index("{", end)
        assert not text[end:body].strip()
        out[called.group(1)] = text[called.end():end - 1], text[body:_closed(text, body, "{}")]
    return out

"""Buffer loads that count on the resource's end to stop them: a raw buffer's bounds
check takes the vector offset and leaves the scalar one out, so a step that may pass
the end has to be in the vector offset.  Read from the sources (no GPU needed): what
such a load brings past the end is masked afterwards, so no result shows it."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "turboquant-pro_amd", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip")))


def calls(text, name):
    """The argument lists of the calls of `name`, split at their own commas."""
    for m in re.finditer(re.escape(name) + r"\(", text):
        depth, args, start = 1, [], m.end()
        for i in range(m.end(), len(text)):
            depth += {"(": 1, "[": 1, "{": 1, ")": -1, "]": -1, "}": -1}.get(text[i], 0)
            if depth == 0 or (depth == 1 and text[i] == ","):
                args.append(" ".join(text[start:i].split()))
                start = i + 1
            if depth == 0:
                break
        yield args


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_loads_into_lds_are_checked_whole(path):
    """The key and value tiles: rows past the last key lie behind the resource's end."""
    with open(path) as f:
        text = f.read()
    for args in calls(text, "__builtin_amdgcn_raw_ptr_buffer_load_lds"):
        assert len(args) == 7, args
        assert args[4] == "0", f"{os.path.basename(path)}: scalar offset {args[4]} past the check"


def test_the_tiles_load_that_way():
    text = open(os.path.join(CSRC, "tqk_attn.hip")).read()
    assert len(list(calls(text, "__builtin_amdgcn_raw_ptr_buffer_load_lds"))) == 3


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_loads_from_registers_steps_are_checked(path):
    """A constant step of a register load, as through a side-list that ends inside
    it, is no scalar offset either."""
    with open(path) as f:
        text = f.read()
    for bits in ("b32", "b64", "b96", "b128"):
        for args in calls(text, "__builtin_amdgcn_raw_buffer_load_" + bits):
            assert len(args) == 4, args
            assert args[2] == "0" or not args[2].isdigit(), f"{os.path.basename(path)}: scalar offset {args[2]}"

"""Stores of more than 8 bytes through a buffer descriptor keep their whole offset in a vector register (no GPU needed): behind one with part of it in a scalar register the
compiler lets the next instruction write the registers that the data still leave from, and zeros have been stored."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "recpulse_amd", "csrc")


def arguments(text, at):
    """The arguments of the call whose opening parenthesis is at text[at]."""
    depth, start, found = 0, at + 1, []
    for i in range(at, len(text)):
        c = text[i]
        if c in "([{":
            depth += 1
        elif c in ")]}":
            depth -= 1
            if depth == 0:
                return found + [text[start:i].strip()]
        elif c == "," and depth == 1:
            found.append(text[start:i].strip())
            start = i + 1
    raise AssertionError("a call without an end")


def test_wide_stores_have_no_scalar_offset():
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*"))):
        text = re.sub(r"//[^\n]*", "", open(path).read()) if path.endswith((".h", ".hip")) else ""
        for call in re.finditer(r"raw_(?:ptr_)?buffer_store_b(?:96|128)\s*\(", text):
            seen += 1
            assert arguments(text, call.end() - 1)[3] == "0", f"{os.path.basename(path)}: a 16-byte store with a scalar offset"
        assert not re.search(r"buffer_store_dwordx[34]", text), f"{os.path.basename(path)}: a 16-byte store in assembly, which this test does not read"
    assert seen >= 5

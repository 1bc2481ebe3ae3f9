"""The Swift shim is not compiled here.  What can be said of its sources without a compiler: which entry points they call, with how many
arguments, and that arrays' sizes are looked at before any of them is taken from an array."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def read(*path):
    with open(os.path.join(ROOT, *path)) as f:
        return f.read()


def arguments(text, at):
    """Top-level arguments of the call whose opening bracket is text[at]."""
    depth, parts, quoted = 0, 1, False
    for i in range(at, len(text)):
        c = text[i]
        quoted ^= c == '"'
        if quoted:
            continue
        depth += c in "([{"
        depth -= c in ")]}"
        parts += c == "," and depth == 1
        if depth == 0:
            return parts if text[at + 1:i].strip() not in ("", "void") else 0
    raise AssertionError("a bracket is not closed")


def test_calls_have_the_arguments_that_the_header_declares():
    header = re.sub(r"/\*.*?\*/", "", read("include", "kvhip.h"), flags=re.S)
    declared = {m[1]: arguments(header, m.end() - 1) for m in re.finditer(r"\b(kvhip_\w+)\(", header)}
    folder = os.path.join("mlx-swift-lm_amd", "swift", "Sources", "KVHIP")
    called = 0
    for name in os.listdir(os.path.join(ROOT, folder)):
        text = re.sub(r"//.*", "", read(folder, name))
        for m in re.finditer(r"\b(kvhip_\w+)\(", text):
            if m[1] in declared:
                assert arguments(text, m.end() - 1) == declared[m[1]], (name, m[1])
                called += 1
    assert called > 30


def test_recurrent_calls_look_at_their_arrays():
    text = read("mlx-swift-lm_amd", "swift", "Sources", "KVHIP", "HIPRecurrent.swift")
    for call, arrays in (("kvhip_short_convolution", ["weight.shape", "bias.shape ==", "window.shape =="]),
                         ("kvhip_gated_delta(", ["a.shape ==", "b.shape ==", "aLog.shape ==", "aLog.kvhipDType ==", "dtBias.kvhipDType ==",
                                                 "deltaState.shape ==", "q.shape == sk"]),
                         ("kvhip_reorder_rows", ["$0.shape[0] == rows"]), ("try check(kvhip_beam_select", ["s.count == 3", "$0.shape == [s[0], s[1]]"])):
        for array in arrays:
            assert 0 <= text.find(array) < text.find(call), (call, array)

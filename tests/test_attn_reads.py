"""The attention kernels mask reads past a cache's end by the buffer's range
check, which covers a lane's own offset but not the scalar offset of the
instruction: an offset that varies by slot has to be in the former.  This test
reads every buffer load and LDS-DMA of fgm_attn.hip and wants a scalar offset of
zero.  (A V cache whose slots are not a multiple of 16 was once read up to three
groups of slots past its end, which no result shows.)"""
from __future__ import annotations

import os
import re

SRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "fastgemma_amd", "csrc", "fgm_attn.hip")


def calls(text: str, name: str) -> list[list[str]]:
    """The argument lists of every call of a function whose name `name` matches."""
    found = []
    for m in re.finditer(rf"\b(?:{name})\(", text):
        depth, args, at = 1, [""], m.end()
        while depth:
            ch = text[at]
            depth += {"(": 1, "{": 1, "[": 1, ")": -1, "}": -1, "]": -1}.get(ch, 0)
            if depth == 1 and ch == ",":
                args.append("")
            elif depth:
                args[-1] += ch
            at += 1
        found.append([a.strip() for a in args])
    return found


def test_calls_are_taken_apart():
    assert calls("x = f(a, g(b, c), {1, 2}); h(0); f(k[i, j], 3)", "f") == [["a", "g(b, c)", "{1, 2}"], ["k[i, j]", "3"]]


def test_attention_reads_have_no_scalar_offset():
    text = re.sub(r"//[^\n]*", "", open(SRC).read())
    loads = calls(text, r"buf_load_\w+") + calls(text, r"dma(?:4|16)(?:<\w+>)?")
    assert len(loads) >= 18
    bad = [a for a in loads if a[-1] != "0"]
    assert not bad, bad

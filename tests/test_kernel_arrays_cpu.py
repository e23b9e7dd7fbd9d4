"""Loops of the kernels' sources stay inside the local arrays that they index (read from the text: an index behind an
array's end has no defined result, and what a compiler makes of it today need not be what the next one does)."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "multi_lora_amd" / "csrc"
SOURCES = sorted(p for p in CSRC.rglob("*") if p.suffix in (".h", ".hip", ".cpp"))
ARRAY = re.compile(r"\b(?:float|int|uint8_t|uint32_t|bool|u32x4|f32x4|raw)\s+((?:\w+(?:\[[^\]]*\])+(?:\s*=\s*\{\})?,?\s*)+);")
LOOP = re.compile(r"\bfor \(int (\w+) = (\w+); \1 < (\d+); (?:\+\+\1|\1 \+= (\d+))\)")


def clean(text):
    """The text without comments and preprocessor lines, lengths kept."""
    blank = lambda m: re.sub(r"[^\n]", " ", m.group())  # noqa: E731
    return re.sub(r"//[^\n]*|/\*.*?\*/|^[ \t]*#[^\n]*", blank, text, flags=re.S | re.M)


def match(text, at, pair):
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == pair[0]) - (text[i] == pair[1])
        if depth == 0:
            return i
    raise ValueError("unbalanced")


def statement_end(text, at):
    """One past the statement that begins at ``at``: a block, a loop or condition with its own, or up to the semicolon."""
    at += len(text[at:]) - len(text[at:].lstrip())
    if text[at] == "{":
        return match(text, at, "{}") + 1
    head = re.match(r"(?:for|while|if(?: constexpr)?) \(", text[at:])
    if head:
        end = statement_end(text, match(text, at + head.end() - 1, "()") + 1)
        after = re.match(r"\s*else\b", text[end:])
        return statement_end(text, end + after.end()) if after else end
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] in "({[") - (text[i] in ")}]")
        if text[i] == ";" and depth == 0:
            return i + 1
    raise ValueError("no end")


def scopes(text):
    """For every declared array of a literal first dimension: (name, size, from, to) of the block it lives in."""
    out, stack = [], []
    starts = {m.start(): m for m in ARRAY.finditer(text)}
    for i, c in enumerate(text):
        if c == "{":
            stack.append(match(text, i, "{}"))
        elif c == "}" and stack:
            stack.pop()
        if i in starts and stack:
            for name, size in re.findall(r"(\w+)\[([^\]]*)\]", re.sub(r"\]\[[^\]]*", "]", starts[i].group(1)).replace("]]", "]")):
                out.append((name, int(size) if size.isdigit() else None, i, stack[-1]))
    return out


def overruns(text):
    text = clean(text)
    arrays, found = scopes(text), []
    for loop in LOOP.finditer(text):
        var, bound = loop.group(1), int(loop.group(3))
        body = text[loop.end():statement_end(text, loop.end())]
        for name in set(re.findall(rf"(?<![\w.>])(\w+)\[{var}\]", body)):
            seen = [a for a in arrays if a[0] == name and a[2] <= loop.start() <= a[3]]
            if seen and seen[-1][1] is not None and seen[-1][1] < bound:
                found.append(f"{name}[{seen[-1][1]}] in a loop to {bound}, line {text[:loop.start()].count(chr(10)) + 1}")
    return found


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_loops_end_with_their_arrays(path):
    assert overruns(path.read_text()) == []


def test_a_loop_that_goes_on_is_found():
    fine = "void f(int s) { float p[8]; for (int i = 0; i < 8; ++i) p[i] = s; { float p[16]; for (int i = 0; i < 16; ++i) { if (s) p[i] = 0; } } %s }"
    assert overruns(fine % "") == []
    for more in ("for (int i = 0; i < 16; ++i) p[i] = 0;", "if (s) {\n for (int i = 0; i < 9; ++i) if (i < s) p[i] = 0; }",
                 "for (int i = 0; i < 10; i += 2) { s += p[i]; }"):
        assert len(overruns(fine % more)) == 1

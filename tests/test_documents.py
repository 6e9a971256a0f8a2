"""The documents' code: every fence that opens closes, Python blocks parse, and no heading lies in one."""

from __future__ import annotations

import ast
import os

import pytest

from conftest import REPO


def blocks(text):
    """(language, lines) of the fenced blocks; a fence that names a language inside a block, or a block
    without an end, is an error."""
    out, language, inside = [], None, []
    for at, line in enumerate(text.split("\n"), 1):
        if line.startswith("```"):
            if language is None:
                language, inside = line[3:].strip(), []
            else:
                assert line.strip() == "```", f"line {at}: a block opens inside another"
                out.append((language, inside))
                language = None
        elif language is not None:
            inside.append(line)
    assert language is None, "the last block has no end"
    return out


@pytest.mark.parametrize("name", ["README.md", "INTEGRATION.md", "DESIGN.md"])
def test_fences_and_python_blocks(name):
    with open(os.path.join(REPO, name), encoding="utf-8") as f:
        text = f.read()
    found = blocks(text)
    for language, lines in found:
        assert not any(line.startswith(("## ", "### ")) for line in lines), lines[:3]
        if language == "python":
            ast.parse("\n".join(lines))
    # What is left are the headings: one title, and no code among them.
    left = text
    for language, lines in found:
        left = left.replace("```" + language + "\n" + "\n".join(lines) + "\n```", "", 1)
    assert sum(line.startswith("# ") for line in left.split("\n")) == 1

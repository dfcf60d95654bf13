"""Kernels that start while the one before them drains (launch_chained in csrc/typed.cuh) may read what that one wrote behind their wait only, and by
plain loads: the compiler takes __ldg and loads through `const ... *__restrict__` for loads of memory that nobody writes while the kernel runs, and may
move them above the wait.  Such a move shows on a GPU by chance, so this reads the sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "project-currennt-public_b200", "csrc")


def _functions(text):
    """name -> head and body of every function of device code"""
    text = re.sub(r"//[^\n]*", "", text)
    out = {}
    for m in re.finditer(r"__(?:global|device)__", text):
        brace = text.find("{", m.end())
        semicolon = text.find(";", m.end())
        if brace < 0 or (0 <= semicolon < brace):
            continue
        head = text[m.start():brace]
        names = re.findall(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\s*\([^()]*(?:\([^()]*\)[^()]*)*\)", "", head))
        if not names:
            continue
        depth, at = 0, brace
        while True:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
            if depth == 0:
                break
        out[names[0]] = text[m.start():at]
    return out


def _chained(text):
    return set(re.findall(r"launch_chained\(\s*(\w+)", re.sub(r"//[^\n]*", "", text)))


FILES = [f for f in sorted(glob.glob(os.path.join(CSRC, "*.cu"))) if "launch_chained(" in open(f).read()]


def test_there_are_such_files():
    assert {os.path.basename(f) for f in FILES} >= {"embedding.cu", "gradient_norm.cu", "block_norm_back.cu"}


@pytest.mark.parametrize("path", FILES, ids=[os.path.basename(f) for f in FILES])
def test_chained_kernels_read_by_plain_loads(path):
    text = open(path).read()
    functions = _functions(text)
    reached, todo = set(), _chained(text)
    assert todo and todo <= set(functions)
    while todo:
        name = todo.pop()
        reached.add(name)
        todo |= {n for n in functions if n not in reached and re.search(r"\b%s\b\s*(?:<[^;()]*>)?\s*\(" % n, functions[name])}
    for name in reached:
        body = functions[name]
        if name in _chained(text):
            assert "grid_wait()" in body, name
        assert "__ldg(" not in body, name
        assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", body), name


@pytest.mark.parametrize("path,kernel", [("logprob.cu", "logprob_backward_kernel"), ("block_norm.cu", "block_norm_few_kernel"), ("block_norm.cu", "block_norm_forward_kernel"),
                                         ("block_norm_back.cu", "block_norm_backward_kernel"), ("gradient_norm.cu", "clip_kernel")])
def test_what_may_be_in_place_is_not_declared_apart(path, kernel):
    """the header lets outputs of these take the place of an input: a __restrict__ of the tensors' type would promise that they do not"""
    head = _functions(open(os.path.join(CSRC, path)).read())[kernel].split("{", 1)[0]
    assert not re.search(r"\bT\s*\*\s*__restrict__", head)

"""The scan-path language model example, end to end: it learns, and every
bracket it writes fits the string before it."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("scan_lm", os.path.join(ROOT, "examples", "scan_lm.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.gpu
def test_scan_lm_example():
    ex = _example()
    first, last, text = ex.main(steps=60)
    assert last < 0.95 * first  # the brackets' frequencies, from a uniform start
    assert len(text) == 43
    stack = []
    for c in text:
        if c in "([":
            stack.append(c)
        elif c == ".":
            assert not stack
        else:
            assert stack and stack.pop() + c in ("()", "[]")


def test_scan_lm_grammar_mask():
    ex = _example()
    assert ex.allowed_next([], "cpu").tolist() == [True, False, True, False, True]
    assert ex.allowed_next([0, 2], "cpu").tolist() == [True, False, True, True, False]
    assert ex.allowed_next([0, 2, 3], "cpu").tolist() == [True, True, True, False, False]

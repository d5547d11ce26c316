"""Every translation unit has its own device error word (common.cuh), so
gfn_get_device_error has to read the word of each unit whose kernels can set it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "manifold_b200", "csrc")
SHARED = ("common.cuh", "umma.cuh")  # define the waits; using one is what sets the word


def _text(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def _own_sources(unit):
    todo, seen = [unit], []
    while todo:
        name = todo.pop()
        if name in seen or name in SHARED or not os.path.exists(os.path.join(CSRC, name)):
            continue
        seen.append(name)
        todo += re.findall(r'#include "([^"]+)"', _text(name))
    return seen


def test_every_unit_that_can_set_its_error_word_is_read():
    units = re.search(r"^SRC := (.*)$", _text("Makefile"), re.M).group(1).split()
    reader = _text("gfn_b200.cu")
    body = reader[reader.index("int gfn_get_device_error("):]
    body = body[:body.index("\n}\n")]
    setting = [u for u in units if any(re.search(r"\b(gfn_flag_error|mbar_wait\w*)\(", _text(s)) for s in _own_sources(u))]
    assert {"norm.cu", "gated_scan.cu", "logits.cu", "layered.cu"} <= set(setting)
    for u in setting:
        name = os.path.splitext(u)[0]
        call = "gfn_unit_error_word(" if name == "gfn_b200" else f"error_word_{name}("
        assert call in body, f"{u} can set its device error word, gfn_get_device_error does not read it"

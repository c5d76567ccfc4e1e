"""The assembly main loops of the big tiles of dense products: what a statement does to registers is what it tells the
compiler, for every one of them."""
import importlib.util
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("gen_products", os.path.join(ROOT, "awesome-cute_amd", "csrc", "gen_products.py"))
gen = importlib.util.module_from_spec(spec)
spec.loader.exec_module(gen)
SHAPES = [(type, layout, rb) for type in gen.TYPES for layout in ("rows", "b", "both") for rb in (5, 6, 7, 8)]


def operands(text):
    """(assembly, outputs, tied, inputs, clobbers) of a statement as the compiler reads it"""
    body, outs, ins, clobbers = re.split(r"\n    : ", text)
    lines = [re.search(r'"(.*?)\\n\\t"', l).group(1) for l in body.splitlines() if l.startswith('    "')]
    constraints = re.findall(r'"([=+]?)\{([^}]*)\}"', outs)
    return (lines, [r for kind, r in constraints if kind == "="], [r for kind, r in constraints if kind == "+"],
            re.findall(r'"\{([^}]*)\}"', ins), re.findall(r'"([^"]*)"', clobbers))


@pytest.mark.parametrize("type,layout,rb", SHAPES)
def test_what_is_written_is_told(type, layout, rb):
    text = gen.statement(gen.Shape(layout, rb), gen.TYPES[type])
    lines, outs, ties, ins, clobbers = operands(text)
    assert {"scc", "memory"} < set(clobbers)
    gen.check_operands(lines, outs, ties, ins, clobbers)
    # the accumulators, all of them and nothing else
    assert set().union(*map(gen.registers, outs)) == {f"a{n}" for n in range(32 * rb)}
    written = set()
    for line in lines:  # (found another way: the first register of everything but loads into LDS, compares and branches)
        name = line.split()[0]
        if not name.endswith(":") and not name.startswith(("buffer_", "s_cmp", "s_cbranch", "s_branch", "s_wait", "s_nop", "s_barrier")):
            written |= gen.registers(line.split()[1].rstrip(","))
    told = set().union(*map(gen.registers, outs + ties + clobbers)) | {"m0"}
    assert written <= told and not written & set().union(*map(gen.registers, ins))


def test_what_is_not_told_is_noticed():
    for type, layout, rb in SHAPES[::3]:
        lines, outs, ties, ins, clobbers = operands(gen.statement(gen.Shape(layout, rb), gen.TYPES[type]))
        for at in (0, 1):
            with pytest.raises(AssertionError):
                gen.check_operands(lines, outs[:at] + outs[at + 1:], ties, ins, clobbers)
            with pytest.raises(AssertionError):
                gen.check_operands(lines, outs, ties[:at] + ties[at + 1:], ins, clobbers)
            with pytest.raises(AssertionError):
                gen.check_operands(lines, outs, ties, ins[:at] + ins[at + 1:], clobbers)
            with pytest.raises(AssertionError):
                gen.check_operands(lines, outs, ties, ins, clobbers[:at] + clobbers[at + 1:])
        with pytest.raises(AssertionError):
            gen.check_operands(lines, outs, ties, ins + ["v5"], clobbers)
        with pytest.raises(AssertionError):
            gen.check_operands(lines + ["v_mov_b32 v5, 0"], outs, ties, ins, clobbers)
        with pytest.raises(AssertionError):
            gen.check_operands(lines + ["s_mov_b32 s90, 0"], outs, ties, ins, clobbers)


def test_registers_of_operands():
    assert gen.registers("v[4:7]") == {"v4", "v5", "v6", "v7"} and gen.registers("s40") == {"s40"}
    assert gen.registers("m0") == {"m0"} and gen.registers("0x400") == set() and gen.registers("offset:512") == set()

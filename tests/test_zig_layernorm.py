"""zig/src/ops/layernorm.zig as text (no Zig toolchain exists here): what it calls is declared, with as many
arguments, and tensors are told apart as the handle {ptr, idx, class} asks (src/core/graph.zig:34-41): an
index counts within its class, so a weight and an input may have the same one."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TEXT = open(os.path.join(ROOT, "zig", "src", "ops", "layernorm.zig")).read()
DECLS = open(os.path.join(ROOT, "include", "kernel_decls.h")).read()


def arguments(text):
    return len([a for a in re.split(r",(?![^(]*\))", text) if a.strip()])


def test_launchers_and_size_functions_are_called_as_declared():
    calls = re.findall(r"core\.invoke\(core\.kernels\.(\w+), key, \.\{(.*?)\}\);", TEXT, re.S)
    assert [c[0] for c in calls] == ["layernorm_ij_j", "layernorm_ij_j_reverse"]
    for stem, args in calls:
        declared = re.search(rf"launch_{stem}_r32\((.*?)\);", DECLS, re.S).group(1)
        assert arguments(args) == arguments(declared), stem
    for name, args in re.findall(r"dev\.(mp\w+)\(([^)]*)\)", TEXT):
        declared = re.search(rf"EXTERN_C len_t {name}\((.*?)\);", DECLS).group(1)
        assert arguments(args) == arguments(declared), name


def test_tensors_are_compared_by_the_whole_handle():
    compared = [line for line in TEXT.splitlines() if re.search(r"\.(idx|ptr|class)\s*[!=]=", line)]
    assert compared and all(".ptr ==" in c and ".idx ==" in c and ".class ==" in c for c in compared), compared


def test_operands_that_share_a_gradient_are_refused():
    """One launch writes the three gradients: x, the gain and the bias must be different tensors."""
    forward = TEXT[TEXT.index("pub fn forward_impl"):TEXT.index("pub fn reverse")]
    for a, b in (("x", "gain"), ("x", "bias"), ("gain", "bias")):
        assert f"std.debug.assert(!same({a}, {b}));" in forward, (a, b)

"""Every direct global-to-LDS load that the library's sources issue from asm is
one whose scalar operands the scalar unit has written one instruction before: the
compiler does not insert the wait states of M0 and of a vector-written base there."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cortexmind_amd", "csrc")


def sources():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".hip", ".hpp")):
            with open(os.path.join(CSRC, name)) as f:
                yield name, re.sub(r"//[^\n]*", "", f.read())


def test_asm_loads_begin_with_the_scalar_move():
    asm = [(n, "".join(re.findall(r"\"([^\"]*)\"", m.group(1)))) for n, text in sources()
           for m in re.finditer(r"asm\s+(?:volatile\s*)?\(((?:\s*\"[^\"]*\")+)", text) if "load_lds" in m.group(1)]
    assert asm
    for name, code in asm:
        steps = [c.strip() for c in code.replace("\\t", " ").split("\\n")]
        for i, c in enumerate(steps):
            if "load_lds" in c:
                base = re.search(r"(%\d)\s*$", c)
                assert i > 0 and base and steps[i - 1].startswith(f"s_mov_b64 {base.group(1)},"), (name, code)


def test_no_load_outside_asm():
    """(The builtin would have the compiler wait for every load before each LDS read.)"""
    for name, text in sources():
        assert not re.search(r"__builtin_amdgcn_(global|raw_buffer|raw_ptr_buffer|struct_buffer)\w*load\w*lds", text), name

"""What the inline assembly of the HIP sources tells the compiler about itself."""
import os
import re

import pytest

from llm_training_amd import _build

SOURCES = sorted(f for f in os.listdir(_build.CSRC) if f.endswith((".hip", ".h")))
# scalar instructions that leave SCC alone; every other one is taken to write it
KEEPS_SCC = {"s_mov_b32", "s_mov_b64", "s_nop", "s_waitcnt", "s_barrier", "s_setprio", "s_sleep"}


def statements(text):
    """The asm statements of a source, comments taken out, each up to its closing parenthesis."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"\basm\s*(?:volatile\s*)?\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += {"(": 1, ")": -1}.get(c, 0)
            i += 1
        yield text[m.start():i]


@pytest.mark.parametrize("src", SOURCES)
def test_scalar_arithmetic_names_scc(src):
    """A scalar comparison that the compiler keeps across a statement would be lost otherwise."""
    for s in statements((_build.CSRC / src).read_text()):
        writes = set(re.findall(r"\bs_[a-z0-9_]+", s)) - KEEPS_SCC
        assert not writes or '"scc"' in s, (src, sorted(writes), s[:200])


def test_statements_are_found():
    text = 'asm volatile("s_add_u32 m0, %0, 4\\n\\t(" : : "s"(f(x)) : "memory"); // asm("s_sub_u32")\nasm("v_exp_f32 %0, %1" : "=v"(a) : "v"(b));'
    got = list(statements(text))
    assert len(got) == 2 and got[0].endswith('"memory")') and "s_sub_u32" not in "".join(got)
    assert len(list(statements((_build.CSRC / "flash_attn_kernels.h").read_text()))) > 20

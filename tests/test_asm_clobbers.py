"""Registers that inline assembly writes behind the compiler's back.

Read from the kernels' sources: an asm statement that changes the condition code
names it as written, exec is put back as it was found, and m0, which the compiler
reserves and refuses to be told of, is set by each statement that reads it."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mega-moe-td_amd", "csrc")


def statements():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h"))):
        text = open(path).read()
        for m in re.finditer(r"\basm volatile\(", text):
            depth, end, quoted = 1, m.end(), False
            while depth:
                c = text[end]
                quoted ^= c == '"'
                depth += 0 if quoted else (c == "(") - (c == ")")
                end += 1
            body = text[m.end():end - 1]
            code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', re.split(r'"\s*:', body)[0] + '"'))
            yield f"{os.path.basename(path)}:{text.count(chr(10), 0, m.start()) + 1}", code, body[body.rindex(":") + 1:]


@pytest.mark.parametrize("where,code,clobbers", [pytest.param(*s, id=s[0]) for s in statements()])
def test_asm_declares_what_it_writes(where, code, clobbers):
    lines = [line.split(None, 1) for line in code.replace("\\t", "").split("\\n") if line.strip()]
    written = {(op, rest.split(",")[0].strip()) for op, rest in lines if op.startswith("s_") and not op.startswith(("s_nop", "s_waitcnt"))}
    if "_lds_" in code:  # a copy to the address in m0
        assert "s_mov_b32 m0, %" in code and code.index("s_mov_b32 m0, %") < code.index("_lds_")
    if any(re.match(r"s_(and|or|xor|not|add|sub|lsh|cmp|bfe)", op) for op, _ in written):
        assert '"scc"' in clobbers
    if any(reg == "exec" for _, reg in written) or "saveexec" in code:
        kept = re.match(r"s_(?:mov_b64|and_saveexec_b64|or_saveexec_b64) (%\d)(?:, exec)?", code.replace("\\t", ""))
        back = re.search(r"s_mov_b64 exec, (%\d)$", code)
        assert kept and back and kept[1] == back[1]


def test_statements_are_found():
    found = list(statements())
    assert len(found) > 10 and sum("m0" in code for _, code, _ in found) >= 5

"""Properties of the kernels' sources that no run would show."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCES = sorted(p for e in ("h", "hip", "cpp") for p in glob.glob(os.path.join(ROOT, "omegalax_amd", "csrc", "*." + e)))


def asm_statements():
    """(file, line, template, clobbers) of every inline assembly statement."""
    for path in SOURCES:
        text = open(path).read()
        for m in re.finditer(r"\basm\s+volatile\s*\(", text):
            depth, at, quoted = 1, m.end(), False
            while depth:
                c = text[at]
                quoted ^= c == '"'
                depth += 0 if quoted else (c == "(") - (c == ")")
                at += 1
            body = text[m.end():at - 1]
            template = "".join(re.findall(r'"([^"]*)"', re.match(r'(\s*"[^"]*")+', body).group(0)))
            rest = body[re.match(r'(\s*"[^"]*")+', body).end():]
            rest = re.sub(r"\([^()]*(\([^()]*(\([^()]*\)[^()]*)*\)[^()]*)*\)", "", rest)  # operands' expressions
            parts = rest.replace("::", ": :").split(":")
            clobbers = re.findall(r'"([^"]*)"', parts[3]) if len(parts) > 3 else []
            yield os.path.basename(path), text.count("\n", 0, m.start()) + 1, template, clobbers


def test_inline_assembly_names_what_it_overwrites():
    """The compiler keeps values of its own in m0 and scc, and over a statement that does not name
    them as overwritten it may keep them there."""
    seen = 0
    for name, line, template, clobbers in asm_statements():
        for op in re.split(r"\\[nt]|;", template):
            words = op.replace(",", " ").split()
            if len(words) < 2:
                continue
            if words[1] == "m0":
                seen += 1
                assert "m0" in clobbers, f"{name}:{line} writes m0"
            if re.match(r"s_(add|sub|and|or|xor|lsh|cmp)", words[0]):
                assert "scc" in clobbers, f"{name}:{line} writes scc"
    assert seen >= 4

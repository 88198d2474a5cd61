"""What the inline assembly of the kernels leaves behind, read from the sources."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "airframe_amd", "csrc")


def statements():
    """(file, text) of every asm statement of the kernels' sources."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        with open(path) as f:
            text = f.read()
        for m in re.finditer(r"\basm\s*(?:volatile\s*)?\(", text):
            depth, i, quoted = 1, m.end(), False
            while depth:
                c = text[i]
                if c == '"' and text[i - 1] != "\\":
                    quoted = not quoted
                elif not quoted:
                    depth += (c == "(") - (c == ")")
                i += 1
            yield os.path.basename(path), text[m.end():i - 1]


def test_m0_is_put_back():
    """The compiler may hold a value of its own in M0: a statement that writes it saves it first and restores it
    last."""
    writes = [(f, s) for f, s in statements() if re.search(r"\bm0\s*,", s)]
    assert writes
    for f, s in writes:
        lines = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', s.split(":")[0])).split("\\n\\t")
        assert re.fullmatch(r"s_mov_b32 (%\d), m0", lines[0]) and lines[-1] == "s_mov_b32 m0, " + lines[0].split()[1][:-1], (f, s)

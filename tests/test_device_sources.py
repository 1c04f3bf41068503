"""Rules of the device sources that no run can show: a breach works until the compiler's register
allocation happens to change."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _asm_blocks():
    for path in sorted(glob.glob(os.path.join(ROOT, "fastermoe_amd", "csrc", "*"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"\basm\s+volatile\s*\((.*?)\)\s*;", text, flags=re.S):
            yield os.path.basename(path), m.group(1)


def test_inline_asm_names_the_special_registers_it_writes():
    """m0 (the LDS address of a direct-to-LDS load) and scc (the result of scalar compares and additions) in the
    clobber list of every asm statement that changes them."""
    seen = 0
    for name, body in _asm_blocks():
        strings = re.findall(r'"((?:[^"\\]|\\.)*)"', body)
        code = [line.strip() for s in strings for line in re.split(r"\\n(?:\\t)?", s)]
        if any(re.match(r"s_\w+\s+m0\b", line) for line in code):
            seen += 1
            assert "m0" in strings, f"{name}: {body}"
        if any(re.match(r"s_(cmp|add|sub|and|or|lshl|lshr)\w*\s", line) for line in code):
            assert "scc" in strings, f"{name}: {body}"
    assert seen >= 3


def test_the_profile_covers_every_launch_of_a_product():
    """Where a file's launches open the profile's scopes themselves, none comes ahead of its function's scope: a product of two launches would be reported with
    the time of one and the work of both."""
    seen = 0
    for name in ("gemm_any.hip", "gemm_kernel.hpp", "gemm_unaligned.hip"):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "fastermoe_amd", "csrc", name)).read())
        for m in re.finditer("<<<", text):
            start = max(f.start() for f in re.finditer(r"^[a-z][^\n;=]*\)\s*\{$", text[:m.start()], flags=re.M))   # its function's first line
            assert re.search(r"ProfileScope", text[start:m.start()]), f"{name}: {text[start:m.start()].splitlines()[0]}"
            seen += 1
    assert seen >= 4

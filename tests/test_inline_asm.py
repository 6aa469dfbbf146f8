"""Inline assembly in the kernels declares what it writes behind its operands:
a statement that sets m0 names it as clobbered, and one that fills LDS by DMA
names memory too, so that the compiler neither keeps a value of its own in m0
nor moves an LDS read across the fill."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "light-rocm-runtime_amd", "csrc")


def statements():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        with open(path) as f:
            text = f.read()
        for m in re.finditer(r"\basm\s+volatile\s*\((.*?)\);", text, re.S):
            yield f"{os.path.basename(path)}:{text.count(chr(10), 0, m.start()) + 1}", m.group(1)


def test_clobbers_are_declared():
    seen = 0
    for where, body in statements():
        code = re.split(r'"\s*:', body, maxsplit=1)[0]
        clobbers = body.rsplit(":", 1)[-1] if body.count(":") >= 3 else ""
        if re.search(r"\b[sv]_\w+ m0\b", code):
            seen += 1
            assert '"m0"' in clobbers, where
        if "global_load_lds" in code or "s_waitcnt" in code or "s_barrier" in code:
            seen += 1
            assert '"memory"' in clobbers, where
    assert seen >= 8


def test_transfers_wait_for_what_they_read():
    """One wait state between the write of m0 and the transfer that reads it, in every form; five where its address is
    in scalar registers too, which a vector instruction may have written right before."""
    seen = 0
    for where, body in statements():
        code, operands = re.split(r'"\s*:', body, maxsplit=1)
        if "global_load_lds" not in code:
            continue
        m = re.search(r"s_mov_b32 m0, %\d\\n\\ts_nop (\d+)\\n\\tglobal_load_lds_dwordx4 %\d, (off|%\d)", code)
        assert m, where
        scalars = re.findall(r'"s"\s*\(', operands)
        assert len(scalars) == (1 if m.group(2) == "off" else 2), where
        assert int(m.group(1)) >= (0 if m.group(2) == "off" else 4), where
        seen += 1
    assert seen >= 5

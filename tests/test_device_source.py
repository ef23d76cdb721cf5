"""Rules of the device sources that no run can show."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lfm2-w9100-rust_amd", "csrc")


def statements(path):
    """The inline-assembly statements of a source."""
    src = re.sub(r"//[^\n]*", "", open(path).read())
    return [src[m.start():src.index(";\n", m.start())] for m in re.finditer(r"\basm\b(?: volatile)?\s*\(", src)]


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h"))),
                         ids=os.path.basename)
def test_assembly_that_uses_m0_names_it(path):
    """A load into shared memory takes its place from M0, which the compiler uses as well: it
    has to see it as an operand, and no statement may write it unseen."""
    for s in statements(path):
        if "_lds_" in s or "lds " in s:
            assert '"{m0}"' in s, s
        assert not re.search(r"\bs_\w+ m0\b", s), s

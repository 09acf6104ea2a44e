"""Rules of the attention kernels' source that no run without a fault can show (CPU)."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-minimaxh3_b200", "csrc")


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_waits_that_a_warp_leaves_on_have_one_verdict():
    """A bounded wait that gives up does so for its whole warp: where lanes took their own verdicts,
    those that stayed would vote and access TMEM without the others, and never return. Single lanes
    (the product issuers), and drains whose verdict nothing reads, may wait by themselves."""
    helper = re.search(r"bool mbar_wait_warp\([^)]*\) \{(.*?)\n\}", _code("common.cuh"), re.S)
    assert helper and re.search(r"return __all_sync\(0xFFFFFFFFu, mbar_wait\(", helper.group(1))
    code = _code("sparse_attention.cu")
    issuer = code.index("constexpr uint32_t kIdescS")
    softmax = code.index("const int row_in = (warp & 3) * 32 + lane;")
    assert 0 < issuer < softmax
    for part in (code[:issuer], code[softmax:]):
        lone = [m for m in re.findall(r"\bmbar_wait\([^;]*;", part) if "kErrSpDrain" not in m]
        assert not lone, lone
    assert len(re.findall(r"\bmbar_wait_warp\(", code[softmax:])) >= 3

"""Source checks of the tensor-core kernels: a warp executes its tensor-memory loads
together.  No GPU needed."""

import pathlib
import re


def _loops(text):
    """The bodies of the for-loops of a source file, innermost ones too."""
    for m in re.finditer(r"\bfor \(", text):
        i, depth = m.end(), 1
        while depth:
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        while text[i].isspace():
            i += 1
        if text[i] != "{":
            continue
        j, depth = i + 1, 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[j], 0)
            j += 1
        yield text[i:j]


def test_a_warp_is_together_before_it_loads_tensor_memory():
    # tcgen05.ld is executed by a whole warp at once.  Lanes without a row leave a trip
    # of such a loop early, so the warp has to meet again before the next trip's load.
    found = 0
    csrc = pathlib.Path(__file__).resolve().parents[1] / "theria_b200" / "csrc"
    for path in sorted(csrc.glob("*.cuh")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for body in _loops(text):
            early = re.search(r"if \((!store|!live|!row_ok|t >= Tq[^{};]*)\) continue;", body)
            load = body.find("tc::tmem_ld")
            if early is None or load < 0 or body.count("for (", 0, load):
                continue
            found += 1
            assert "__syncwarp();" in body[:load], (path.name, body[:200])
    assert found >= 8

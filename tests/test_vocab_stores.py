"""The vocabulary's kernels store past the caches where a launcher asks for it and not elsewhere, on the CPU: the gfx950 code objects
that `__graft_entry__.build()` compiled in this tree from its own sources are disassembled.  Results that the next kernel finds in
the caches are stored the default way, and both instantiations of every family exist."""
import os
import re

import pytest

from tests.test_streaming_stores import BUILD, _kernels, _tools

# (object, family, the last template arguments of the instantiations that stream, of those that do not)
FAMILIES = [
    ("kernels_embedding.hip.o", "k_embedding", r"Lb1EEE", r"Lb0EEE"),
    ("kernels_embedding.hip.o", "k_embed_sum", r"Lb0ELb1EEE", r"Lb[01]ELb0EEE"),  # ADD, NT
    ("kernels_distill.hip.o", "k_distill_grad", r"Lb1EEE", r"Lb0EEE"),
    ("kernels_adjust_logits.hip.o", "k_adjust", r"Lb1EEE", r"Lb0EEE"),
]


@pytest.mark.parametrize("obj,family,stream,default", FAMILIES)
def test_stores_follow_their_policy(obj, family, stream, default, tmp_path):
    path = os.path.join(BUILD, obj)
    if not os.path.exists(path) or not _tools():
        pytest.skip("build objects or ROCm LLVM tools missing (run __graft_entry__.build() first)")
    kernels = {n: b for n, b in _kernels(path, str(tmp_path)).items() if re.match(rf"_ZN3mpy\d+{family}I", n)}
    assert kernels
    seen = {True: 0, False: 0}
    for name, body in kernels.items():
        streams = re.search(stream, name) is not None
        assert streams or re.search(default, name), name
        held = any(re.search(r"\bglobal_store_\w+\b.*\bnt\b", line) for line in body.splitlines())
        assert held == streams, f"{name}: streaming {streams}, but a streaming store {held}"
        seen[streams] += 1
    assert seen[True] and seen[False], seen

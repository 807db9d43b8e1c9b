"""What the compiler made of the sequence kernels: none may keep values in scratch memory (one that did returned a wrong count;
the cause was not found, so none is let through).  Reads the metadata of the object file that this repository builds."""
import os
import re

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJ = os.path.join(REPO, "marl_amd", "csrc", "build", "seq_kernels.o")


def _numbers(blob, key):
    """The values of `key` in the kernels' metadata (MessagePack: small ones in the byte behind the key, larger ones behind a tag)."""
    out = []
    for m in re.finditer(re.escape(key) + rb"(?=[\x00-\x7f\xcc-\xcf])", blob):
        tag = blob[m.end()]
        out.append(tag if tag < 0x80 else int.from_bytes(blob[m.end() + 1:m.end() + 1 + (1 << (tag - 0xcc))], "big"))
    return out


@pytest.mark.skipif(not os.path.isfile(OBJ), reason="not built here")
def test_no_kernel_uses_scratch_memory():
    blob = open(OBJ, "rb").read()
    scratch, spilled, waves = (_numbers(blob, k) for k in (b".private_segment_fixed_size", b".vgpr_spill_count", b".wavefront_size"))
    assert len(scratch) == len(spilled) == len(waves) > 100 and set(waves) == {64}
    assert set(scratch) == {0} and set(spilled) == {0}

"""The argument structures that the bindings pack byte by byte have the layout of the C header (compiled here by the C compiler)."""
import os
import shutil
import struct
import subprocess

import pytest

from segk import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# field -> its place among the packed values, in order
ATTENTION = {"N": 0, "dtype": 6, "causal": 7, "scale": 8, "q": 9, "k": 13, "v": 17, "out": 21, "lse": 25, "out_rest": 26, "mask": 27,
             "mask_n": 28, "mask_k": 31, "key_mask": 32, "key_mask_k": 34, "dout": 35, "dq": 39, "dk": 40, "dv": 41}
ROTARY = {"N": 0, "dtype": 5, "q": 6, "k": 10, "q_out": 14, "k_out": 15, "q_weight": 16, "k_weight": 17, "positions": 18, "pos_dtype": 19,
          "pos_n": 20, "pos_a": 22, "axes": 23, "section": 24, "inv_freq": 28, "norm": 29, "interleaved": 30, "eps": 31, "dq": 32,
          "dk": 36, "dq_weight": 40, "dk_weight": 41}


def offsets(packer):
    """Byte offsets of a native-alignment struct's values."""
    codes = []
    count = ""
    for c in packer.format.lstrip("@"):
        if c.isdigit():
            count += c
        else:
            codes += [c] * int(count or 1)
            count = ""
    at, res = 0, []
    for c in codes:
        size = struct.calcsize(c)
        at = (at + size - 1) // size * size
        res.append(at)
        at += size
    return res


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_layouts(tmp_path):
    kinds = (("segk_attention_args", ATTENTION, _lib.ATTENTION_ARGS), ("segk_qk_norm_rotary_args", ROTARY, _lib.QK_NORM_ROTARY_ARGS))
    lines = []
    for name, fields, _ in kinds:
        for f in list(fields) + ["workspace"]:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, f))
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
    source = tmp_path / "layout.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "segk.h"\nint main(void) {\n%s\nreturn 0;\n}\n' % "\n".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(tmp_path / "layout")])
    found = iter(map(int, subprocess.check_output([str(tmp_path / "layout")], text=True).split()))
    for name, fields, packer in kinds:
        packed = offsets(packer)
        for f, i in fields.items():
            assert next(found) == packed[i], (name, f)
        assert next(found) == packer.size, (name, "workspace")
        assert next(found) == packer.size + _lib.WORKSPACE_ARGS.size, name

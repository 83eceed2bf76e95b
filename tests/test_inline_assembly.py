"""What inline assembly writes beside its outputs is declared to the compiler, which sets m0 for accesses of its own and may keep it."""
import glob
import os
import re

import liteform_ae_amd

STATEMENT = re.compile(r"\basm\b(?:\s+volatile)?\s*\((.*?)\);", re.S)


def statements():
    for path in sorted(glob.glob(os.path.join(os.path.dirname(liteform_ae_amd.__file__), "csrc", "*"))):
        for text in STATEMENT.findall(open(path).read()):
            yield os.path.basename(path), text


def test_m0_is_declared_as_written():
    writes = [(path, text) for path, text in statements() if re.search(r'"[^"]*\bs_\w+ m0,', text)]
    assert writes
    for path, text in writes:
        assert '"m0"' in text.rsplit(":", 1)[1], f"{path}: {text}"

"""The C entries of the training-step operators: every declared symbol is exported and bound."""
import os
import re

from bit_reproducible_training_amd import _lib

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol():
    names = set()
    for header in ("repro_adamw.h", "repro_norm.h", "repro_loss.h"):
        with open(os.path.join(REPO, "include", header)) as f:
            text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
        names |= set(re.findall(r"\b(rg_[a-z0-9_]+)\s*\(", text))
    assert names and names == set(_lib._MODEL_SIGNATURES)
    for name in names:
        assert hasattr(_lib.lib, name), name

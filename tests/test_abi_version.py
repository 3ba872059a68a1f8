"""The header's version changes with every struct and signature in it: both are pinned together, so that changing one without
the other fails here and not in a caller that was built against the other."""
import hashlib
import os
import re

import pytest

from maester_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PINNED = (10300, "38e6b1eec68731c8")


def _declarations():
    """The header without comments, its version and white space."""
    text = open(os.path.join(ROOT, "include", "maester_attn.h")).read()
    version = int(re.search(r"#define\s+MA_ABI_VERSION\s+(\d+)", text).group(1))
    text = re.sub(r"/\*.*?\*/", " ", text, flags=re.S)
    text = re.sub(r"#define\s+MA_ABI_VERSION.*", "", text)
    return version, re.sub(r"\s+", " ", text).strip()


def test_version_and_declarations():
    version, text = _declarations()
    digest = hashlib.sha256(text.encode()).hexdigest()[:16]
    assert (version, digest) == PINNED, "a struct or a signature changed: raise MA_ABI_VERSION, then pin both here"


def test_the_binding_and_the_guide_name_the_headers_version():
    version, _ = _declarations()
    assert _lib.MA_ABI_VERSION == version == _lib.lib().ma_version()
    guide = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    assert {int(v) for v in re.findall(r"ma_version\(\) == (\d+)", guide)} == {version}


def test_a_library_of_another_header_is_refused(monkeypatch):
    # the last version before log-probabilities took the parts of a gradient: their arguments stood in other places
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "MA_ABI_VERSION", 10200)
    with pytest.raises(RuntimeError, match="10200"):
        _lib.lib()

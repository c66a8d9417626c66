"""Libraries whose entry points take other arguments than this binding hands them are not loaded."""
import hashlib
import os
import re
import subprocess

import pytest

from openattention_amd import _build, lib

HDR = os.path.join(os.path.dirname(_build.HERE), "include", "openattention_amd.h")


def prototypes():
    """The header's structs and functions, without comments and line breaks"""
    text = open(HDR).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    text = text[text.index("OA_ENOSPC"):]
    return re.sub(r"\s+", " ", text)


# what the entry points of each version and revision looked like
KNOWN = {(9, 1): "1ad4bfc334b66865"}


def test_a_changed_entry_point_comes_with_a_changed_revision():
    """A prototype that changes while version and revision stay would let an older library be called by it."""
    digest = hashlib.sha256(prototypes().encode()).hexdigest()[:16]
    assert KNOWN.get((lib.ABI_VERSION, lib.ABI_REVISION)) == digest, f"prototypes changed: raise the revision, for {digest}"


@pytest.mark.parametrize("revision,want", [(None, "lacks oa_abi_revision"), (0, "revision 0"), (99, "revision 99")])
def test_a_library_of_another_revision_is_refused(revision, want, tmp_path, monkeypatch):
    """Also where it has this version and every other entry point, whose arguments may be others."""
    body = f"int oa_abi_version(void) {{ return {lib.ABI_VERSION}; }}\n"
    if revision is not None:
        body += f"int oa_abi_revision(void) {{ return {revision}; }}\n"
    body += "".join(f"int {n}(void) {{ return 0; }}\n" for n in lib.SIGNATURES if n not in ("oa_abi_version", "oa_abi_revision"))
    src, so = tmp_path / "old.c", tmp_path / "old.so"
    src.write_text(body)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
    monkeypatch.setattr(_build, "lib_path", lambda: str(so))
    monkeypatch.setattr(lib, "_LIB", None)
    with pytest.raises(RuntimeError, match=want) as e:
        lib.load()
    assert "rebuild it" in str(e.value)

"""CPU test: the fingerprint of the kernel sources covers all that the library is compiled from."""

import re
from pathlib import Path

from b200_attention_b200 import build, registry


def fingerprinted(monkeypatch):
    seen = set()
    read = Path.read_bytes
    with monkeypatch.context() as m:
        m.setattr(Path, "read_bytes", lambda self: seen.add(self.resolve()) or read(self))
        registry.source_closure_sha256(registry.KERNELS[0])
    return seen


def test_every_included_file_counts(monkeypatch):
    seen = fingerprinted(monkeypatch)
    assert seen >= {p.resolve() for p in build.CORE_SOURCES}
    for path in seen:
        for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', path.read_text(), re.M):
            assert (path.parent / name).resolve() in seen, f"{path.name} includes {name}"


def test_a_change_anywhere_changes_the_fingerprint(monkeypatch):
    before = registry.source_closure_sha256(registry.KERNELS[0])
    read = Path.read_bytes
    for name in ("plan.h", "attn_plan_sm100.cu", "attn_fwd_sm100.cu", "b200_attention.h"):
        with monkeypatch.context() as m:
            m.setattr(Path, "read_bytes", lambda self: read(self) + (b"//" if self.name == name else b""))
            assert registry.source_closure_sha256(registry.KERNELS[0]) != before, name
    assert registry.source_closure_sha256(registry.KERNELS[0]) == before

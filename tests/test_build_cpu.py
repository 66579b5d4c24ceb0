"""What the build rebuilds: every object when any header that a source includes changes."""

from __future__ import annotations

import importlib.util
import re
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "cute-moe-train_b200"


def _build_module():
    spec = importlib.util.spec_from_file_location("mgf_build_under_test", PKG / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _included(source: Path, roots: list[Path], seen: set[Path]) -> set[Path]:
    """Headers of this repository that `source` includes, directly or through others."""
    for name in re.findall(r'^#include "([^"]+)"', source.read_text(), re.M):
        for root in roots:
            path = root / name
            if path.exists() and path not in seen:
                seen.add(path)
                _included(path, roots, seen)
    return seen


@pytest.mark.parametrize("part", ["build_lib", "build_ops"])
def test_every_included_header_is_a_dependency(part, monkeypatch):
    b = _build_module()
    calls = []
    monkeypatch.setattr(b, "_objects", lambda srcs, headers, *a: calls.append((srcs, headers)) or [])
    monkeypatch.setattr(b, "_newer", lambda *a: False)
    getattr(b, part)()
    ((srcs, headers),) = calls
    assert srcs
    for src in srcs:
        missing = _included(src, [b.CSRC, b.INCLUDE], set()) - set(headers)
        assert not missing, f"{src.name}: {sorted(p.name for p in missing)}"

"""CPU: the entry points whose argument types are declared (lib.Entry) match the header's prototypes, argument by argument."""

import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def _letters(params: str) -> str:
    out = ""
    for p in params.split(","):
        p = p.strip()
        out += "p" if "*" in p else "q" if "ng_i64" in p or "ng_u64" in p else "f" if p.startswith("float") else "i"
        assert out[-1] != "i" or re.match(r"int\s+\w+$", p), p
    return out


def test_declared_types_match_the_header():
    from ngram_amd import build, embed, kvcache, tree

    if not build.lib_path().exists():
        build.build()
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "ngram_amd.h").read_text(), flags=re.S)
    entries = [e for m in (embed, kvcache, tree) for e in m._entries()]
    assert len(entries) == 8
    for e in entries:
        params = re.search(r"^\s*int\s+%s\s*\(([^;]*?)\)\s*;" % e.name, text, flags=re.M | re.S).group(1)
        assert e.types + "p" == _letters(params), e.name


def test_a_failing_call_raises(monkeypatch):
    from ngram_amd import lib

    monkeypatch.setattr(lib, "_device", lambda: 0)
    monkeypatch.setattr(lib, "_stream", lambda d: 0)
    e = lib.Entry(name="ng_tree_mask", types="piip")
    with pytest.raises(RuntimeError, match="ng_tree_mask returned -1"):
        e(0, None, 1, 65, None)  # refused before anything is launched

"""CPU: the beam step's entry point with its exponent in 64 bits: its declared types are the header's, and what it refuses it
refuses before anything is launched."""

import ctypes
import math
import re

import pytest
from test_entries import ROOT

from ngram_amd import beam, build, lib


@pytest.fixture
def step(monkeypatch):
    if not build.lib_path().exists():
        build.build()
    monkeypatch.setattr(lib, "_device", lambda: 0)
    monkeypatch.setattr(lib, "_stream", lambda d: 0)
    return beam._step()


def test_declared_types_match_the_header(step):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "ngram_amd.h").read_text(), flags=re.S)
    params = re.search(r"^\s*int\s+%s\s*\(([^;]*?)\)\s*;" % step.name, text, flags=re.M | re.S).group(1)
    kinds = [("p", r".*\*.*"), ("q", r"ng_i64 \w+"), ("d", r"double \w+"), ("i", r"int \w+")]
    letters = [next(k for k, form in kinds if re.fullmatch(form, p.strip(), re.S)) for p in params.split(",")]
    assert step.types + "p" == "".join(letters) and step.types.count("d") == 1
    assert step.fn.argtypes[step.types.index("d")] is ctypes.c_double


def test_exponents_refused_before_a_launch(step):
    """Null addresses throughout: a call that went on would fault."""
    def call(B, alpha, lengths):
        step(0, None, 18, 9, 0, None, lengths, 4, None, B, 2, 9, 2, -1, -1, alpha, None, None, None, None, None, None)

    call(0, 0.6, 64)
    call(0, 1e300, 64)
    for alpha, lengths in ((-1.0, 64), (math.nan, 64), (math.inf, 64), (0.6, None)):
        for B in (0, 1):
            with pytest.raises(RuntimeError, match="returned -1"):
                call(B, alpha, lengths)


@pytest.mark.parametrize("V", [1, 8192, 8193, 50257, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, 1056831, 3_000_000, 1 << 25, (1 << 25) + 1])
def test_stated_limits(step, V):
    """Sizes are taken up to the limits that the header and the refusal state, and no further."""
    chunks = -(-V // 8192)
    for B, W in ((0, 1), (1, 1), (1, 128), (1, 129), (1 << 24, 1), ((1 << 24) + 1, 1), (1 << 24, 128), (1 << 20, 64), (4, 8)):
        for K in (1, 2, 4, 5, 63, 64, 100, 126, 127, 128, 129):
            within = (B <= 1 << 24 and W <= 128 and K <= 128 and V <= 1 << 25 and K <= W * V and K * chunks <= 16384
                      and B * W * chunks < 1 << 31)
            size = lib.Lib().size("ng_beam_work", B, W, V, K)
            assert (size >= 0) == within, (B, W, V, K)
            if not within:
                with pytest.raises(ValueError, match="16384"):
                    beam._work(B, W, V, K)

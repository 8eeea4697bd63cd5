"""CPU: the decoding operators' entry points (beam, pages, sparse): their declared argument types match the header, and what
they refuse they refuse before anything is launched."""

import re

import pytest

from test_entries import ROOT, _letters

from ngram_amd import beam, build, pages, sparse
from ngram_amd.lib import Lib


@pytest.fixture(scope="module")
def library():
    if not build.lib_path().exists():
        build.build()
    return Lib()


@pytest.fixture
def host(monkeypatch):
    from ngram_amd import lib

    monkeypatch.setattr(lib, "_device", lambda: 0)
    monkeypatch.setattr(lib, "_stream", lambda d: 0)


def test_declared_types_match_the_header(library):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "ngram_amd.h").read_text(), flags=re.S)
    entries = [e for m in (beam, pages, sparse) for e in m._entries()]
    assert len(entries) == 10
    for e in entries:
        params = re.search(r"^\s*int\s+%s\s*\(([^;]*?)\)\s*;" % e.name, text, flags=re.M | re.S).group(1)
        assert e.types + "p" == _letters(params), e.name


def test_sizes(library):
    assert library.size("ng_beam_work", 1, 4, 50257, 4) > 0
    assert library.size("ng_beam_work", 0, 1, 1, 1) >= 0
    for bad in ((-1, 1, 9, 1), (1, 0, 9, 1), (1, 129, 9, 1), (1, 1, 0, 1), (1, 1, 9, 0), (1, 1, 9, 10), (1, 2, 900, 129),
                (1, 1, (1 << 25) + 1, 1), (1, 1, 1 << 21, 128)):
        assert library.size("ng_beam_work", *bad) == -1, bad
    assert library.size("ng_pool_state", 33) == (3 * 33 + 2 + 1) * 4
    assert library.size("ng_pool_state", 0) == library.size("ng_pool_state", 1 << 31) == -1
    assert library.size("ng_pool_fork_work", 1024, 5) == 0 and library.size("ng_pool_fork_work", 1025, 5) == 1025 * 6 * 4
    assert library.size("ng_pool_fork_work", 1, 1 << 27) == -1
    assert library.size("ng_pool_room_work", 2, 1, 16) == (3 * 4 + 2) * 4
    assert library.size("ng_pool_room_work", 2, 18, 16) == (3 * 6 + 2) * 4
    for bad in ((1, 0, 16), (1, 1, 8), (1, 1, 48), (1, 1 << 30, 16), (1 << 27, 100, 16)):
        assert library.size("ng_pool_room_work", *bad) == -1, bad
    assert library.size("ng_pool_move_work", 4, 9) == 52 and library.size("ng_pool_move_work", 0, 9) == -1
    assert library.size("ng_sparse_work", 1, 1, 8, 4, 128, 320, 16, 32) > 0
    for bad in ((1, 0, 8, 4, 128, 320, 16, 32), (1, 1, 0, 4, 128, 320, 16, 32), (1, 1, 8, 0, 128, 320, 16, 32),
                (1, 1, 8, 4, 257, 320, 16, 32), (1, 1, 8, 4, 128, 32769, 16, 32), (1, 1, 8, 4, 128, 320, 24, 32),
                (1, 1, 8, 4, 128, 320, 16, 1025), (1, 1, 8, 4, 128, 320, 16, 0)):
        assert library.size("ng_sparse_work", *bad) == -1, bad


def test_refused_before_a_launch(library, host):
    """Null addresses throughout: a call that went on would fault."""
    step, gather = beam._entries()

    def beam_step(B=1, W=2, V=9, K=2, dtype=0, lsize=4, end=-1, pad=-1, alpha=0.0, finished=None, out_lengths=None):
        step(0, None, 18, 9, dtype, None, None, lsize, finished, B, W, V, K, end, pad, alpha, None, None, None, None, out_lengths, None)

    beam_step(B=0)
    for bad in (dict(W=0), dict(K=19), dict(dtype=3), dict(alpha=-1.0), dict(alpha=1.0), dict(finished=64), dict(finished=64, pad=9),
                dict(out_lengths=64), dict(alpha=float("nan"))):
        with pytest.raises(RuntimeError, match="returned -1"):
            beam_step(**bad)
    gather(0, None, 0, 0, 4, None, 0, None)
    with pytest.raises(RuntimeError, match="returned -1"):
        gather(0, None, 0, 0, 4, None, -1, None)
    clear, hold, fork, room, move, copy = pages._entries()
    for call in (lambda: clear(0, None, 0), lambda: hold(0, None, 5, None, 4, -1, 4), lambda: fork(0, None, 5, None, 4, 1, 0, None, None, None),
                 lambda: room(0, None, 5, None, 4, 1, 4, None, None, 0, None, None, None, None, 16, 1, 64, 0, None, None),
                 lambda: room(0, None, 5, None, 4, 1, 4, None, None, 1, None, None, None, None, 16, 1, 300, 0, None, None),
                 lambda: move(0, None, 5, None, None, None, None, None, None, 5, None, None, None, None, 64, 16, 1, 64, 0, None, 4, 1,
                              4, None, None),
                 lambda: copy(0, None, None, None, None, None, 5, None, None, None, None, None, 5, 17, 1, 64, 0, None, None, 1),
                 lambda: copy(0, None, None, None, None, None, 5, None, None, None, None, None, 5, 16, 1, 64, 0, None, None, -1)):
        with pytest.raises(RuntimeError, match="returned -1"):
            call()
    hold(0, None, 5, None, 4, 0, 4)
    fork(0, None, 5, None, 4, 0, 4, None, None, None)
    copy(0, None, None, None, None, None, 5, None, None, None, None, None, 5, 16, 1, 64, 2, None, None, 0)
    bounds, attend = sparse._entries()
    bounds(0, None, None, 5, 16, 1, 64, 2, None, 4, 4, None, 0, 1, None)
    for bad in ((0, 16, 1, 64, 2), (5, 20, 1, 64, 2), (5, 16, 0, 64, 2), (5, 16, 1, 0, 2), (5, 16, 1, 64, 4), (5, 16, 1, 64, 0)):
        with pytest.raises(RuntimeError, match="returned -1"):
            bounds(0, None, None, *bad, None, 4, 4, None, 1, 1, None)

    def sparse_attention(B=1, T=1, codes=2, qtype=1, keep=4, first=1, last=1, page=16, width=9):
        attend(0, None, 64, 64, 64, qtype, None, None, None, None, None, 5, page, codes, None, 9, width, None, None, B, T, 1, 1, 64, keep,
               first, last, 1.0, None, None, None, None)

    sparse_attention(B=0)
    for bad in (dict(T=0), dict(codes=0), dict(qtype=2), dict(qtype=0), dict(keep=0), dict(last=0), dict(first=-1), dict(first=4),
                dict(page=15), dict(width=0), dict(codes=5)):
        with pytest.raises(RuntimeError, match="returned -1"):
            sparse_attention(**bad)

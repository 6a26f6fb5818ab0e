"""The build entry compiles whatever is there already: a library that is newer than its sources may
still be older than the flags it is to be built with."""
import __graft_entry__
from abmarl_amd import _native
from oracle import oracle


def test_build_compiles_what_is_built(monkeypatch):
    calls = []
    monkeypatch.setattr(_native, 'build', lambda force=False, **kw: calls.append(('engine', force)))
    monkeypatch.setattr(_native, 'build_learn', lambda force=False, **kw: calls.append(('learn', force)))
    monkeypatch.setattr(oracle, 'build', lambda *a, **kw: calls.append(('oracle', True)))
    __graft_entry__.build()
    assert calls == [('engine', True), ('learn', True), ('oracle', True)]

"""What the smoke run reaches: every serving operator, and drafts that are refused."""

from __future__ import annotations

import pytest

from cuda_b200 import paged, speculative

pytestmark = pytest.mark.gpu


def test_smoke_reaches_every_operator_and_refuses_drafts(monkeypatch):
    import __graft_entry__ as entry

    called, dropped = set(), []
    for name in ("extend", "append", "attend", "fork", "truncate", "release", "compact", "copy_pages"):
        def wrapped(self, *args, _name=name, _method=getattr(paged.PagedCache, name), **kwargs):
            called.add(_name)
            if _name == "truncate":
                dropped.append(int(args[0].sum()))
            return _method(self, *args, **kwargs)

        monkeypatch.setattr(paged.PagedCache, name, wrapped)
    verify, rows = speculative.verify, []

    def counted(*args, **kwargs):
        rows.append(verify(*args, **kwargs))
        return rows[-1]

    monkeypatch.setattr(speculative, "verify", counted)
    entry.serve_smoke()
    assert called == {"extend", "append", "attend", "fork", "truncate", "release", "compact", "copy_pages"}
    assert rows and sum(dropped) > 0
    assert any(int((accepted < emitted.shape[1] - 1).sum()) for accepted, emitted in rows)

"""GPU test of the decode layer's command from an empty cache."""

import pytest
import torch

import decode_opt_b200 as dg
from decode_opt_b200 import decode_layer as dl

pytestmark = pytest.mark.gpu


def test_from_an_empty_cache(monkeypatch, capsys):
    """No two requests have a page in common at the end."""
    tables, real = [], dg.build_block_tables
    monkeypatch.setattr(dg, "build_block_tables", lambda *a, **kw: tables.append((a[3], a[4])) or real(*a, **kw))
    assert dl.main(["--requests", "7", "--context", "0", "--steps", "40", "--hidden", "512", "--heads", "4", "--kv-heads",
                    "2", "--page-size", "2"]) == 0
    assert "us a step" in capsys.readouterr().out
    table, page = tables[0]
    held = table[:, :(40 + 4) // page].flatten().tolist()      # 4 steps before the timed ones
    assert len(set(held)) == len(held)

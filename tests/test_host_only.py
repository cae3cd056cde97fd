"""Tests whose pointers are made up must not run where a card would follow them."""
from pathlib import Path

import pytest

import conftest

HERE = Path(__file__).resolve().parent


class Item:
    def __init__(self, path):
        self.fspath, self.markers = path, []

    def add_marker(self, m):
        self.markers.append(m.name)


@pytest.mark.parametrize("card", [True, False])
def test_made_up_addresses_and_cards(card, monkeypatch):
    monkeypatch.setattr(conftest, "card_present", lambda: card)
    # every file that has such an address
    made_up = sorted(p.name for p in HERE.glob("test_*.py") if "0x7f0000000000" in p.read_text() and p != Path(__file__))
    assert "test_mx4_args.py" in made_up
    items = [Item(HERE / n) for n in made_up] + [Item(HERE / "test_abi.py")]
    conftest.pytest_collection_modifyitems(None, items)
    assert [i.markers for i in items] == [["skip"] if card else []] * len(made_up) + [[]]

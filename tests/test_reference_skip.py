"""The comparison with the reference's compiled kernels is left out only where
they can neither be found nor built."""
from __future__ import annotations

import conftest


def test_missing_build_of_sources_at_hand_is_not_skipped(tmp_path, monkeypatch):
    import __graft_entry__

    class Item:
        def __init__(self, name):
            self.name, self.keywords, self.marks = name, (), []

        def add_marker(self, mark):
            self.marks.append(mark)

    def left_out():
        items = [Item("test_reference_family_agrees"), Item("test_other")]
        conftest.pytest_collection_modifyitems(None, items)
        assert items[1].marks == []
        return bool(items[0].marks)

    monkeypatch.setattr(conftest, "ROOT", tmp_path / "repo")
    monkeypatch.setattr(__graft_entry__, "REFERENCE", tmp_path / "sources")
    assert left_out()  # nothing to build from
    family = tmp_path / "sources" / "kernels" / "q4k" / "q4k_family.cu"
    family.parent.mkdir(parents=True)
    family.touch()
    assert not left_out()  # not built, though it could be: the test runs and fails
    family.unlink()
    lib = tmp_path / "repo" / "oracle" / "_ref" / "libq4k_ref.so"
    lib.parent.mkdir(parents=True)
    lib.touch()
    assert not left_out()

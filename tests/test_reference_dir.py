"""Finding the reference's sources: a directory without them counts as absent."""
import os
import sys

from conftest import REPO, reference_dir

sys.path.insert(0, REPO)
import __graft_entry__  # noqa: E402


def test_an_empty_directory_is_no_reference(tmp_path, monkeypatch):
    monkeypatch.setenv("PT_REFERENCE_DIR", str(tmp_path))
    assert reference_dir() is None and __graft_entry__._reference_dir() is None
    os.makedirs(tmp_path / "runtime" / "v21" / "src")
    assert reference_dir() == str(tmp_path) == __graft_entry__._reference_dir()

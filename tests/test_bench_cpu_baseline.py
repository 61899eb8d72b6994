"""bench.py's CPU baseline: what it says without the compiled reference, and that other missing files stay
errors."""
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_without_the_compiled_reference(monkeypatch, tmp_path):
    import bench
    import oracle.cpu
    monkeypatch.setattr(oracle.cpu, "REF_SO", str(tmp_path / "none.so"))
    assert bench.cpu_baseline("model", None) == {"unavailable": "oracle/_ref is not built"}


def test_another_missing_file_is_an_error(monkeypatch, tmp_path):
    import bench
    import oracle.cpu
    so = tmp_path / "ref.so"
    so.write_bytes(b"")
    monkeypatch.setattr(oracle.cpu, "REF_SO", str(so))

    def measure(*a, **k):
        raise FileNotFoundError("model")

    monkeypatch.setattr(bench, "cpu_reference", measure)
    with pytest.raises(FileNotFoundError, match="model"):
        bench.cpu_baseline("model", None)
    monkeypatch.setattr(bench, "cpu_reference", lambda path, x, n: (2.0, 4, 3, 1.5))
    got = bench.cpu_baseline("model", None)
    assert got["value"] == 2.0 and got["cores"] == 4 and "12 samples" in got["sample"]

"""The comparison kernels' build where the reference's sources are absent."""
import os

from oracle import build_ref_gpu


def test_no_sources_means_no_build_not_an_error(tmp_path, monkeypatch):
    monkeypatch.setattr(build_ref_gpu, "OUT", str(tmp_path / "lib.so"))
    assert build_ref_gpu.build(str(tmp_path / "missing")) is None
    os.makedirs(tmp_path / "empty")
    assert build_ref_gpu.build(str(tmp_path / "empty")) is None
    (tmp_path / "lib.so").write_bytes(b"")  # one built elsewhere is taken
    assert build_ref_gpu.build(str(tmp_path / "empty")) == str(tmp_path / "lib.so")

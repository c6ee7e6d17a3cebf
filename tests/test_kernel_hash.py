"""bench.kernel_source_hash: what ties a committed traffic measurement to the machine code it was taken on."""
import os
import shutil

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_hash_covers_the_sources_and_the_flags_they_are_compiled_with(tmp_path, monkeypatch):
    import bench
    csrc = tmp_path / "musev_amd" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    for n in os.listdir(os.path.join(ROOT, "musev_amd", "csrc")):
        if n.endswith((".hip", ".h", ".sh")):
            shutil.copy(os.path.join(ROOT, "musev_amd", "csrc", n), csrc / n)
    shutil.copy(os.path.join(ROOT, "include", "musev_hip.h"), tmp_path / "include")
    here = bench.kernel_source_hash()
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    assert bench.kernel_source_hash() == here
    script = (csrc / "build.sh").read_text()
    for old, new, same in ((" -O3", " -O2", False), (" -packed-fp32-ops", " -other", False), ("mkdir -p $OBJ", "mkdir -p $OBJ  # (objects)", True)):
        assert old in script
        (csrc / "build.sh").write_text(script.replace(old, new))
        assert (bench.kernel_source_hash() == here) == same, new
    (csrc / "build.sh").write_text(script)
    (csrc / "norm.hip").write_text((csrc / "norm.hip").read_text() + "\n")
    assert bench.kernel_source_hash() != here

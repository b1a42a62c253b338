"""CPU: the counters that bench.py prints beside its timings describe the kernels of this tree."""
import os
import shutil

import bench


def test_the_stamp_follows_the_profiled_kernels_alone(tmp_path, monkeypatch):
    shutil.copytree(os.path.join(bench.ROOT, "tsdiff_amd", "csrc"), tmp_path / "tsdiff_amd" / "csrc",
                    ignore=lambda d, names: [n for n in names if not n.endswith((".hip", ".hpp"))])
    shutil.copytree(os.path.join(bench.ROOT, "include"), tmp_path / "include")
    want = bench.kernel_source_sha()
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    assert bench.kernel_source_sha() == want
    csrc = tmp_path / "tsdiff_amd" / "csrc"
    for name in bench.BLOCK_SOURCES:
        assert (csrc / name).exists()
        (csrc / name).write_text("// another kernel")
        assert bench.kernel_source_sha() == want, name
    (csrc / "kernels_combo.hip").write_text("// another kernel")
    assert bench.kernel_source_sha() != want

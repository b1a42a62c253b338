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
    header = tmp_path / "include" / "tsdiff_hip.h"
    header.write_text(header.read_text().replace("/* element types", "/* the element types"))
    assert bench.kernel_source_sha() == want
    (csrc / "kernels_combo.hip").write_text("// another kernel")
    assert bench.kernel_source_sha() != want


def test_the_committed_counters_are_of_this_trees_kernels():
    """a change to a profiled kernel asks for tools/profile_round.sh's counter passes anew; otherwise the bench line would lose
    `traffic` and `mfma_busy` without a word"""
    for name in (bench.PMC_C2, bench.PMC_C5, bench.MFMA_BUSY):
        data, note = bench._stamped(name)
        assert data is not None, note
    for kernel, name in (("forward_mega_kernel<256>", bench.PMC_C2), ("unit_encoder_kernel<256>", bench.PMC_C5),
                         ("cfconv_aggregate_win_kernel<256", bench.PMC_C5)):
        assert bench.pmc_traffic(kernel, name)[0] > 0, kernel
    for label, kernel in (("c2", "forward_mega_kernel<256>"), ("train", "block_bwd_kernel"), ("train", "wgrad_h2_batch_kernel")):
        assert 0 < bench.mfma_busy(label, kernel) < 1, kernel

"""bench.py's hash over the sources of the splat's kernels, in a made-up tree: no GPU needed."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def bench():
    spec = importlib.util.spec_from_file_location("igs_bench_sources", os.path.join(ROOT, "bench.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("line", ['#include "igs_b.h"', '  #  include "igs_b.h"  // a reason', '#include <igs_b.h>', '#include "b.inc"'])
def test_hash_follows_includes_of_includes(bench, tmp_path, monkeypatch, line):
    """A file that only a header includes is among the sources; one that nothing includes is not; a cycle ends."""
    csrc = tmp_path / "igs_amd" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    inner = "b.inc" if "b.inc" in line else "igs_b.h"
    (csrc / "igs_gs2d.hip").write_text('#include <hip/hip_runtime.h>\n#include "igs_hip.h"\nnamespace {\n#include "igs_a.h"\n}\n')
    (csrc / "igs_a.h").write_text(line + "\n")
    (csrc / inner).write_text('#include "igs_a.h"\nint one;\n')
    (csrc / "igs_other.h").write_text("int two;\n")
    (tmp_path / "include" / "igs_hip.h").write_text("int three;\n")
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    before = bench.csrc_sha16()
    (csrc / "igs_other.h").write_text("int changed;\n")
    assert bench.csrc_sha16() == before
    for changed in (csrc / inner, csrc / "igs_a.h", csrc / "igs_gs2d.hip", tmp_path / "include" / "igs_hip.h"):
        text = changed.read_text()
        changed.write_text(text + "// changed\n")
        assert bench.csrc_sha16() != before, changed
        changed.write_text(text)
    assert bench.csrc_sha16() == before

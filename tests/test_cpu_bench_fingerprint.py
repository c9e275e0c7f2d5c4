"""Which sources a counter summary under profiles/ is valid for (bench.kernel_source_fingerprint)."""
import json
import os
import shutil

import bench


def test_the_committed_summaries_are_of_these_kernels():
    prof = os.path.join(bench.ROOT, "profiles")
    for kind in ("traffic", "mfma"):
        prints = [json.load(open(os.path.join(prof, f)))["kernel_sources_sha256"] for f in sorted(os.listdir(prof)) if f.endswith(f"_{kind}.json")
                  and "kernel_sources_sha256" in open(os.path.join(prof, f)).read()]
        assert bench.kernel_source_fingerprint() in prints, kind


def test_sources_of_other_kernels_do_not_count_and_flags_do(tmp_path, monkeypatch):
    csrc = tmp_path / "humanrf_amd" / "csrc"
    shutil.copytree(os.path.join(bench.ROOT, "humanrf_amd", "csrc"), csrc, ignore=shutil.ignore_patterns("_build"))
    before = bench.kernel_source_fingerprint()
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    assert bench.kernel_source_fingerprint() == before
    for name in bench.OTHER_SOURCES:
        with open(csrc / name, "a") as f:
            f.write("// more\n")
    assert bench.kernel_source_fingerprint() == before
    make = (csrc / "Makefile").read_text()
    (csrc / "Makefile").write_text(make.replace("-O3", "-O2"))
    assert bench.kernel_source_fingerprint() != before
    (csrc / "Makefile").write_text(make)
    with open(csrc / "march.hip", "a") as f:
        f.write("// more\n")
    assert bench.kernel_source_fingerprint() != before

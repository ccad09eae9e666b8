"""How the kernels are compiled: the same source has to give the same code."""
from heterofusedkernels_b200 import build


def test_one_compilation_a_translation_unit(monkeypatch):
    """-split-compile cuts a translation unit by the threads that happen to be free, and what is inlined and unrolled changes with
    the cut: the same source gave libraries of 4.6 and of 5.2 MB, one with kernels 5 % slower than the other."""
    seen = []
    monkeypatch.setattr(build, "_run", lambda cmd, *a, **k: seen.append([str(x) for x in cmd]))
    build.build_capi(force=True)
    assert len(seen) == 1 and "arch=compute_100a,code=sm_100a" in seen[0]
    assert not any("split-compile" in x or x in ("-t", "--threads") for x in seen[0])

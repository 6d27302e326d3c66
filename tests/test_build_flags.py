"""How the libraries are compiled."""
from bpt_amd import _build


def test_warnings_of_inline_assembly_are_off_for_one_library_alone(monkeypatch):
    runs = []
    monkeypatch.setattr(_build, "_run", lambda cmd, verbose: runs.append(cmd))
    for build in (_build.build_attn, _build.build_plan, _build.build_score, _build.build_block, _build.build_bias, _build.build_linear):
        build(False)
    quiet = [cmd for cmd in runs if "-Wno-inline-asm" in cmd]
    assert len(runs) == 6 and [cmd[-1] for cmd in quiet] == [_build.LINEAR_SO]
    # no library is built with packed float32 instructions
    assert all("-packed-fp32-ops" in cmd for cmd in runs)

"""Calls of more elements than a launch has threads for are refused before anything is launched (include/bptlinear.h, include/bptbias.h)."""
from bpt_amd import _lib
from test_epilogue_bias_abi import AT, SIZE, linear, ref
from test_score_abi import plan


def test_dropout_of_more_elements_than_threads():
    lib = linear()
    for n, dtype in ((2 ** 36, 0), (2 ** 37, 2), (2 ** 39 + 4096, 0), (2 ** 40, 2)):
        assert lib.bpt_dropout(AT, None, AT, n, 0.5, 0, dtype, None) == SIZE, (n, dtype)


def test_codes_of_more_places_than_threads():
    lib = _lib.bias_lib()
    for entries in (2 ** 30, 2 ** 30 + 7, 2 ** 31):
        p = plan(n_grp_entries=entries)
        for out in (None, plan()):
            assert lib.bpt_bucket_prepare(ref(p), ref(out), AT, AT, 3, 8, 8, 0.1, 0, AT, None) == SIZE, entries

"""CPU checks of the batched serving calls' limits: sizes whose launches the device could not take are refused before
anything is launched."""
import ctypes

import pytest

import cdna4

P = ctypes.c_void_p(64)   # aligned, never dereferenced: validation fails first


@pytest.mark.parametrize("cfg,fits", [
    ((64, 2048, 2048, 2 ** 15, 64, 0, 0, 0), False),          # 2^26 rows: 2^32 threads would join them
    ((64, 2048, 2048, 2 ** 16, 0, 0, 0, 0), False),           # no key at all: rows of zeros are written too
    ((64, 1024, 1, 2 ** 17, 1, 0, 0, 0), False),
    ((64, 1, 1, 2 ** 26 - 4, 1, 0, 0, 0), True),
    ((64, 1, 1, 2 ** 26 - 3, 1, 0, 0, 0), False),
])
def test_shared_rows_fit_the_join(cfg, fits):
    c, info = cdna4.SharedDecodeCfg(*cfg), cdna4.PlanInfo()
    rc = cdna4.lib().cdna4_attn_decode_shared_plan(ctypes.byref(c), cdna4.F16, ctypes.byref(info))
    assert rc == (0 if fits else 1)
    assert (cdna4.decode_shared_workspace_size(c) > 0) == fits
    if not fits:
        assert cdna4.lib().cdna4_attn_decode_shared(P, P, P, P, P, P, P, ctypes.byref(c), cdna4.F16, P, 1 << 62, None) == 1

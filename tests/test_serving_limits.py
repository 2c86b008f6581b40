"""CPU checks of the batched serving calls' limits: sizes whose launches the device could not take are refused before
anything is launched."""
import ctypes

import pytest
import torch

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


def logits_args(**kw):
    a = cdna4.LogitsArgs()
    a.logits, a.out, a.M, a.V, a.logits_stride, a.out_stride = 64, 64, 3, 100, 100, 100
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("dtype,kw,fits", [
    (cdna4.F32, {}, True), (cdna4.F32, dict(M=1, out_stride=104), True), (cdna4.F32, dict(out_stride=104), False),
    (cdna4.F16, {}, False), (cdna4.BF16, dict(logits_stride=200), False), (cdna4.F16, dict(out=4096), True),
])
def test_logits_in_place(dtype, kw, fits):
    """Results over the logits themselves only where each lies where its logit was: a workgroup would overwrite what
    another has yet to read."""
    if fits and torch.cuda.is_available():
        pytest.skip("would be launched on these addresses; in place on the GPU: test_gpu_logits.py")
    rc = cdna4.lib().cdna4_process_logits(ctypes.byref(logits_args(**kw)), dtype, None)
    assert (rc != 1) == fits      # without a GPU the device check is what refuses a valid call


@pytest.mark.parametrize("heads,o_head,fits", [((8, 4), 64, True), ((8, 4), 60, False), ((8, 4), 0, False), ((1, 1), 0, True)])
def test_packed_heads_of_the_output_do_not_overlap(heads, o_head, fits):
    """Heads of O written over each other (an expanded tensor, for instance)."""
    if fits and torch.cuda.is_available():
        pytest.skip("would be launched on these addresses")
    c = cdna4.PackedPrefillCfg(64, *heads, 3, 100, 50, 0, 0)
    s = cdna4.PackedStrides(512, 64, 256, 64, 512, o_head)
    rc = cdna4.lib().cdna4_attn_prefill_packed(P, P, P, None, None, P, P, ctypes.byref(c), ctypes.byref(s), cdna4.F16, None, 0, None)
    assert (rc != 1) == fits

"""CPU checks of the batched serving entry points: exported, and refusing what they do not support before any
GPU work."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import cdna4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p(64)   # aligned, never dereferenced: validation fails first


def test_cdna4_symbols_exported():
    text = open(os.path.join(ROOT, "include", "cdna4_attn.h")).read()
    names = set(re.findall(r"\b(cdna4_[a-z0-9_]+)\s*\(", text))
    out = subprocess.run(["nm", "-D", "--defined-only", cdna4.library_path()], capture_output=True, text=True, check=True).stdout
    assert names <= set(re.findall(r"\bT (cdna4_\w+)", out)), names


def packed(cfg=(64, 8, 4, 3, 100, 50, 0, 0), strides=(512, 64, 256, 64, 512, 64), dtype=cdna4.F16, Q=P, K=P, V=P, Kp=None, Vp=None, O=P, cu=P, ws=None, n=0):
    c, s = cdna4.PackedPrefillCfg(*cfg), cdna4.PackedStrides(*strides)
    return cdna4.lib().cdna4_attn_prefill_packed(Q, K, V, Kp, Vp, O, cu, ctypes.byref(c), ctypes.byref(s), dtype, ws, n, None)


@pytest.mark.parametrize("cfg", [
    (96, 8, 4, 3, 100, 50, 0, 0), (64, 8, 3, 3, 100, 50, 0, 0), (64, 0, 4, 3, 100, 50, 0, 0), (64, 8, 0, 3, 100, 50, 0, 0),
    (64, 8, 4, -1, 100, 50, 0, 0), (64, 8, 4, 3, -1, 50, 0, 0), (64, 8, 4, 3, 100, 101, 0, 0), (64, 8, 4, 3, 100, -1, 0, 0),
    (64, 8, 4, 3, 100, 50, -1, 0), (64, 8, 4, 3, 100, 50, 2 ** 31 - 100, 0)])
def test_packed_refuses_configurations(cfg):
    assert packed(cfg) == 1
    info = cdna4.PlanInfo()
    c = cdna4.PackedPrefillCfg(*cfg)
    if cfg[6] < 2 ** 30:
        assert cdna4.lib().cdna4_attn_prefill_packed_plan(ctypes.byref(c), cdna4.F16, ctypes.byref(info)) == 1


def test_packed_refuses_arguments():
    good = (64, 8, 4, 3, 100, 50, 0, 0)
    pre = (64, 8, 4, 3, 100, 50, 20, 0)
    odd = ctypes.c_void_p(72)
    assert packed(good, dtype=cdna4.F32) == 1 and packed(good, dtype=9) == 1
    for name in ("Q", "K", "V", "O", "cu"):
        assert packed(good, **{name: None}) == 1, name
    for name in ("Q", "K", "V"):
        assert packed(good, **{name: odd}) == 1, name            # 8 bytes off 16
    assert packed(good, O=ctypes.c_void_p(68)) == 1 and packed(good, cu=ctypes.c_void_p(66)) == 1
    assert packed(pre) == 1 and packed(pre, Kp=P) == 1 and packed(pre, Kp=P, Vp=odd) == 1
    assert packed((64, 8, 4, 3, 100, 50, 20, 19), Kp=P, Vp=P) == 1    # rows between heads below the prefix
    for i, bad in ((0, 60), (0, 516), (1, 4), (2, 56), (2, 260), (3, -64), (4, 60), (4, 510), (5, 2)):
        st = [512, 64, 256, 64, 512, 64]
        st[i] = bad
        assert packed(good, strides=st) == 1, (i, bad)
    l = cdna4.lib()
    assert l.cdna4_attn_prefill_packed(P, P, P, None, None, P, P, None, None, cdna4.F16, None, 0, None) == 1
    # nothing to do: no pointer is needed
    assert packed((64, 8, 4, 0, 100, 50, 0, 0), Q=None, K=None, V=None, O=None, cu=None) == 0
    assert packed((64, 8, 4, 3, 0, 0, 0, 0), Q=None, K=None, V=None, O=None, cu=None) == 0


def test_packed_plan():
    for D, dt in ((64, torch.float16), (128, torch.bfloat16)):
        c = cdna4.PackedPrefillCfg(D, 32, 8, 24, 12961, 2048, 0, 0)
        p = cdna4.prefill_packed_plan(c, dt)
        assert p.name == "fa_packed" and p.workspace == cdna4.prefill_packed_workspace_size(c)
        assert (p.workspace > 0) == (D == 128)
        small = cdna4.PackedPrefillCfg(D, 12, 12, 7, 161, 61, 0, 0)
        assert cdna4.prefill_packed_workspace_size(small) == 0
        # a workspace that is too small or misaligned is refused, a missing one is not needed (checked on the GPU)
        for ws, n in ((P, p.workspace - 1), (ctypes.c_void_p(72), p.workspace)) if p.workspace else ():
            assert packed((D, 32, 8, 24, 12961, 2048, 0, 0), (32 * D, D, 8 * D, D, 32 * D, D), ws=ws, n=n) == 1
    with pytest.raises(cdna4.CDNA4Error):
        cdna4.prefill_packed_plan(cdna4.PackedPrefillCfg(64, 8, 3, 1, 10, 0, 0, 0))


@pytest.mark.parametrize("cfg", [
    (64, 8, 4, 3, 100, 50, 2 ** 31 - 100, 0), (64, 8, 4, 3, 2 ** 31 - 1, 50, 0, 0), (64, 8, 4, 3, 100, 50, 20, 19),
    (64, 8, 4, 2 ** 20 + 1, 100, 50, 0, 0), (64, 8, 4, 2 ** 31 - 1, 2 ** 30, 0, 0, 0),
    (128, 1025, 1025, 2 ** 20, 2 ** 20, 0, 0, 0)])
def test_packed_refuses_sizes_past_32_bits(cfg):
    """Key indices, sequences and blocks that 32-bit counters could not hold: the plan and the size refuse what the
    call refuses."""
    info, c = cdna4.PlanInfo(), cdna4.PackedPrefillCfg(*cfg)
    assert cdna4.lib().cdna4_attn_prefill_packed_plan(ctypes.byref(c), cdna4.F16, ctypes.byref(info)) == 1
    assert cdna4.prefill_packed_workspace_size(c) == 0
    row = cfg[1] * cfg[0]
    if cfg[1] == 8:   # the blocks of the last are counted when the device is known
        assert packed(cfg, (row, cfg[0], row, cfg[0], row, cfg[0]), Kp=P, Vp=P) == 1


def test_packed_python_refuses_cpu_tensors():
    x = torch.zeros(10, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        cdna4.prefill_packed(x, x, x, x, torch.zeros(2, dtype=torch.int32), cdna4.PackedPrefillCfg(64, 4, 4, 1, 10, 10, 0, 0))


def logits_args(**kw):
    a = cdna4.LogitsArgs()
    a.logits = a.out = a.history = a.bias_ids = a.bias_values = a.mask = 64
    a.M, a.V, a.logits_stride, a.out_stride = 3, 100, 100, 104
    a.history_max, a.history_stride, a.n_bias, a.mask_stride = 5, 5, 2, 4
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    dict(V=0), dict(V=-1), dict(V=2 ** 31 - 1), dict(M=-1), dict(M=65536), dict(logits_stride=99), dict(out_stride=99),
    dict(history_stride=4), dict(history_max=-1), dict(history_max=2 ** 24 + 1), dict(n_bias=-1), dict(n_bias=8193),
    dict(mask_stride=3), dict(logits=None), dict(out=None), dict(bias_ids=None), dict(bias_values=None), dict(logits=65),
    dict(out=66), dict(history=66), dict(repetition=66), dict(mask=65), dict(prompt_len=63)])
def test_logits_refuses(bad):
    a = logits_args(**bad)
    assert cdna4.lib().cdna4_process_logits(ctypes.byref(a), cdna4.F16, None) == 1


def test_logits_refuses_dtypes_and_null():
    a = logits_args()
    for dt in (cdna4.F64, cdna4.I32, 9, -1):
        assert cdna4.lib().cdna4_process_logits(ctypes.byref(a), dt, None) == 1
    assert cdna4.lib().cdna4_process_logits(None, cdna4.F16, None) == 1
    a = logits_args(logits=66)
    assert cdna4.lib().cdna4_process_logits(ctypes.byref(a), cdna4.F32, None) == 1   # fp32 rows are 4-byte aligned
    a = logits_args(M=0, logits=None, out=None)
    assert cdna4.lib().cdna4_process_logits(ctypes.byref(a), cdna4.F32, None) == 0   # nothing to do


def shared(cfg=(128, 8, 2, 4, 100, 0, 50, 0), dtype=cdna4.F16, q=P, Kp=P, Vp=P, K=P, V=P, lens=P, o=P, ws=P, n=None):
    c = cdna4.SharedDecodeCfg(*cfg)
    if n is None:
        n = cdna4.decode_shared_workspace_size(c)
    return cdna4.lib().cdna4_attn_decode_shared(q, Kp, Vp, K, V, lens, o, ctypes.byref(c), dtype, ws, n, None)


@pytest.mark.parametrize("cfg", [
    (96, 8, 2, 4, 100, 0, 50, 0), (128, 8, 3, 4, 100, 0, 50, 0), (128, 0, 2, 4, 100, 0, 50, 0), (128, 8, 0, 4, 100, 0, 50, 0),
    (128, 8, 2, -1, 100, 0, 50, 0), (128, 8, 2, 4, -1, 0, 50, 0), (128, 8, 2, 4, 100, 99, 50, 0), (128, 8, 2, 4, 100, 0, -1, 0),
    (128, 8, 2, 4, 100, 0, 50, 49), (128, 8, 2, 4, 2 ** 31 - 1, 0, 50, 0), (128, 8, 2, 4, 100, 0, 2 ** 31 - 1, 0),
    (128, 2 ** 20, 1, 2 ** 20, 100, 0, 50, 0)])
def test_shared_refuses_configurations(cfg):
    assert shared(cfg, n=1 << 60) == 1
    assert cdna4.decode_shared_workspace_size(cdna4.SharedDecodeCfg(*cfg)) == 0
    info = cdna4.PlanInfo()
    c = cdna4.SharedDecodeCfg(*cfg)
    assert cdna4.lib().cdna4_attn_decode_shared_plan(ctypes.byref(c), cdna4.F16, ctypes.byref(info)) == 1


def test_shared_refuses_arguments():
    odd = ctypes.c_void_p(72)
    for name in ("q", "Kp", "Vp", "K", "V", "lens", "o", "ws"):
        assert shared(**{name: None}) == 1, name
    for name in ("q", "Kp", "Vp", "K", "V", "ws"):
        assert shared(**{name: odd}) == 1, name
    assert shared(o=ctypes.c_void_p(66)) == 1 and shared(lens=ctypes.c_void_p(66)) == 1
    assert shared(dtype=cdna4.F32) == 1 and shared(dtype=9) == 1
    need = cdna4.decode_shared_workspace_size(cdna4.SharedDecodeCfg(128, 8, 2, 4, 100, 0, 50, 0))
    assert need > 0 and shared(n=need - 1) == 1
    assert shared((128, 8, 2, 0, 100, 0, 50, 0), q=None, o=None, ws=None, n=0) == 0     # nothing to do
    p = cdna4.decode_shared_plan(cdna4.SharedDecodeCfg(128, 32, 8, 64, 8192, 0, 1024, 0))
    assert p.name == "decode_shared" and p.workspace == cdna4.decode_shared_workspace_size(cdna4.SharedDecodeCfg(128, 32, 8, 64, 8192, 0, 1024, 0))
    assert p.grid * 256 < 2 ** 32


CALLER = r"""
#include <cdna3/attention.hpp>
#include <cdna3/runtime/forward.hpp>
using namespace cdna3;
int main() {
    attn::PackedCfg p{64, 8, 4, 3, 100, 50, 0, 0};
    attn::PackedStrides st = attn::packed_strides(p);
    if (st.q_row != 512 || st.kv_row != 256 || st.o_head != 64) return 1;
    const __half* h = nullptr;
    const __hip_bfloat16* b = nullptr;
    if (attn::prefill_packed(h, h, h, (__half*)nullptr, nullptr, p, st) != hipErrorInvalidValue) return 2;
    if (attn::prefill_packed(b, b, b, (__hip_bfloat16*)nullptr, nullptr, p, st, b, b, nullptr, nullptr, 0) != hipErrorInvalidValue) return 3;
    if (attn::prefill_packed_workspace_size(p) != 0) return 4;
    attn::SharedDecodeCfg s{128, 8, 2, 4, 100, 0, 50, 0};
    if (attn::decode_shared_workspace_size(s) == 0) return 5;
    if (attn::decode_shared(h, h, h, h, h, nullptr, (__half*)nullptr, s, nullptr, 0) != hipErrorInvalidValue) return 6;
    if (attn::decode_shared(b, b, b, b, b, nullptr, (__hip_bfloat16*)nullptr, s, nullptr, 0) != hipErrorInvalidValue) return 7;
    runtime::LogitsArgs a{};
    if (runtime::process_logits(a, CDNA4_F16) != hipErrorInvalidValue) return 8;
    return 0;
}
"""


def test_cxx_callers(tmp_path):
    clang = "/opt/rocm/llvm/bin/clang++"
    if not os.path.exists(clang):
        pytest.skip("no clang++")
    src, exe = tmp_path / "caller.cpp", tmp_path / "caller"
    src.write_text(CALLER)
    lib = os.path.dirname(cdna4.library_path())
    r = subprocess.run([clang, "-std=c++17", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"),
                        str(src), "-o", str(exe), "-L" + lib, "-lcdna4_attn", "-Wl,-rpath," + lib, "-L/opt/rocm/lib", "-lamdhip64",
                        "-Wl,-rpath,/opt/rocm/lib"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    assert subprocess.run([str(exe)]).returncode == 0

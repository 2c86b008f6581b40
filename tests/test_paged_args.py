"""CPU checks of the paged cache's and the beams' entry points: exported, refusing what they do not support before any GPU work, and
the MXFP4 reference of the GPU tests."""
import ctypes
import os
import subprocess

import pytest
import torch

import cdna4
from paged_util import GRID, pack, quantise, unpack, values

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p(64)   # aligned, never dereferenced: validation fails first
ODD8, ODD4, ODD2 = ctypes.c_void_p(72), ctypes.c_void_p(68), ctypes.c_void_p(66)
GOOD = dict(D=128, nKVHeads=2, page=64, pages=10, format=0, max_pages=4, table_stride=0)
BAD_CACHES = [dict(D=96), dict(D=0), dict(nKVHeads=0), dict(page=8), dict(page=48), dict(page=512), dict(page=0), dict(page=-16), dict(pages=0),
              dict(format=2), dict(format=-1), dict(max_pages=0), dict(max_pages=2 ** 25), dict(table_stride=3), dict(table_stride=-1),
              dict(nKVHeads=2 ** 17), dict(nKVHeads=2 ** 16, page=256)]


def cache(**kw):
    return cdna4.PagedCache(*{**GOOD, **kw}.values())


def decode(c=None, cfg=(8, 3, 1), dtype=cdna4.F16, q=P, K=P, V=P, tables=P, lens=P, o=P, ws=P, n=None):
    c, f = c or cache(max_pages=400), cdna4.PagedDecodeCfg(*cfg)   # a table of several workgroups per sequence
    n = cdna4.decode_paged_workspace_size(c, f) if n is None else n
    return cdna4.lib().cdna4_attn_decode_paged(q, K, V, tables, lens, o, ctypes.byref(c), ctypes.byref(f), dtype, ws, n, None)


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_caches_are_refused(bad):
    c = cache(**bad)
    cfg = cdna4.PagedDecodeCfg(8 if "nKVHeads" not in bad else max(1, bad["nKVHeads"]), 3, 1)
    assert cdna4.decode_paged_workspace_size(c, cfg) == 0
    assert decode(c, (cfg.nQHeads, 3, 1), n=1 << 60) == 1
    assert append(c) == 1 and reorder(c) == 1


@pytest.mark.parametrize("cfg", [(7, 3, 1), (0, 3, 1), (8, -1, 1), (8, 3, 0), (8, 3, 17), (8, 2 ** 24, 1), (2 ** 20, 2 ** 10, 1), (8, 2 ** 19, 16)])
def test_decode_refuses_configurations(cfg):
    assert decode(cfg=cfg, n=1 << 60) == 1
    c, f, info = cache(), cdna4.PagedDecodeCfg(*cfg), cdna4.PlanInfo()
    assert cdna4.decode_paged_workspace_size(c, f) == 0
    assert cdna4.lib().cdna4_attn_decode_paged_plan(ctypes.byref(c), ctypes.byref(f), cdna4.F16, ctypes.byref(info)) == 1


def test_decode_refuses_arguments():
    for name in ("q", "K", "V", "tables", "lens", "o", "ws"):
        assert decode(**{name: None}) == 1, name
    for name in ("q", "K", "V", "ws"):
        assert decode(**{name: ODD8}) == 1, name
    for name in ("tables", "lens", "o"):
        assert decode(**{name: ODD2}) == 1, name
    assert decode(dtype=cdna4.F32) == 1 and decode(dtype=9) == 1
    need = cdna4.decode_paged_workspace_size(cache(max_pages=400), cdna4.PagedDecodeCfg(8, 3, 1))
    assert need > 0 and decode(n=need - 1) == 1
    assert decode(cfg=(8, 0, 1), q=None, K=None, V=None, tables=None, lens=None, o=None, ws=None, n=0) == 0   # nothing to do
    p = cdna4.decode_paged_plan(cache(max_pages=400), cdna4.PagedDecodeCfg(8, 3, 1))
    assert p.name == "decode_paged" and p.workspace == need and p.waves == 1 and p.grid == p.partials < 2 ** 26


def test_decode_of_short_tables_needs_no_workspace():
    c, f = cache(), cdna4.PagedDecodeCfg(8, 3, 1)
    p = cdna4.decode_paged_plan(c, f)
    assert (p.workspace, p.partials, p.grid, p.waves) == (0, 1, 6, 4) and cdna4.decode_paged_workspace_size(c, f) == 0
    assert decode(c, K=None, ws=None) == 1


def test_decode_refuses_more_keys_than_shares_count():
    c = cache(nKVHeads=8, page=256, max_pages=2 ** 22, pages=2 ** 20)
    for batch, ok in ((1, True), (2 ** 20, False)):
        assert (cdna4.decode_paged_workspace_size(c, cdna4.PagedDecodeCfg(8, batch, 1)) > 0) == ok
    assert decode(c, (8, 2 ** 20, 1), n=1 << 60) == 1


def append(c=None, dtype=cdna4.F16, **kw):
    a = cdna4.AppendArgs()
    for f in ("q", "k", "v", "q_out", "K_pages", "V_pages", "tables", "positions"):
        setattr(a, f, 64)
    a.eps, a.T, a.nQHeads, a.batch, a.max_pos = 1e-6, 3, 8, 3, 0
    for k, v in kw.items():
        setattr(a, k, v)
    c = c or cache()
    return cdna4.lib().cdna4_rope_append_paged(ctypes.byref(a), ctypes.byref(c), dtype, None)


@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(T=2 ** 26), dict(nQHeads=-1), dict(nQHeads=2 ** 20 + 1), dict(batch=0), dict(max_pos=-1), dict(eps=-1e-6), dict(eps=float("nan")),
    dict(cos_tab=64), dict(sin_tab=64), dict(q=None), dict(q_out=None), dict(k=None), dict(v=None), dict(K_pages=None), dict(V_pages=None),
    dict(tables=None), dict(positions=None), dict(q_row=1020), dict(q_row=1026), dict(k_row=252), dict(v_row=258), dict(q_out_row=1000), dict(k_out_row=-256),
    dict(v_out_row=255), dict(q=68), dict(k=66), dict(v=65), dict(q_out=68), dict(k_out=68), dict(v_out=68), dict(q_norm=68), dict(k_norm=68),
    dict(K_pages=72), dict(V_pages=72), dict(cos_tab=72, sin_tab=64), dict(cos_tab=64, sin_tab=72), dict(tables=66), dict(seqs=66), dict(positions=66),
    dict(q_row=2048), dict(k_out=64, k_row=512), dict(v_out=64, v_out_row=512)])
def test_append_refuses(bad):
    """The last ones: an output at its input's address with another row stride."""
    assert append(**bad) == 1


def test_append_refuses_dtypes_and_null():
    for dt in (cdna4.F32, cdna4.F64, cdna4.I32, 9, -1):
        assert append(dtype=dt) == 1
    c = cache()
    assert cdna4.lib().cdna4_rope_append_paged(None, ctypes.byref(c), cdna4.F16, None) == 1
    a = cdna4.AppendArgs()
    assert cdna4.lib().cdna4_rope_append_paged(ctypes.byref(a), None, cdna4.F16, None) == 1
    a.batch = 1
    assert cdna4.lib().cdna4_rope_append_paged(ctypes.byref(a), ctypes.byref(c), cdna4.F16, None) == 0   # no tokens


def reorder(c=None, parents=64, tables=128, lens=192, fresh=256, to=320, lens_to=384, K=64, V=64, rows=3, rows_in=3, layers=1, stride=0):
    c = c or cache()
    return cdna4.lib().cdna4_paged_reorder(parents, tables, lens, fresh, to, lens_to, K, V, ctypes.byref(c), rows, rows_in, layers, stride, None)


@pytest.mark.parametrize("bad", [
    dict(parents=None), dict(tables=None), dict(lens=None), dict(fresh=None), dict(to=None), dict(lens_to=None), dict(K=None), dict(V=None),
    dict(parents=66), dict(to=322), dict(K=72), dict(V=72), dict(rows=-1), dict(rows=65536), dict(rows_in=0), dict(layers=0), dict(layers=4097),
    dict(stride=16), dict(stride=10 * 2 * 64 * 256 + 8), dict(stride=-16), dict(to=128), dict(lens_to=192), dict(lens_to=64)])
def test_reorder_refuses(bad):
    assert reorder(**bad) == 1


def test_reorder_of_nothing():
    assert reorder(parents=None, tables=None, lens=None, fresh=None, to=None, lens_to=None, K=None, V=None, rows=0) == 0


def beam(dtype=cdna4.F16, ws=P, n=1 << 40, **kw):
    a = cdna4.BeamArgs()
    for f in ("logits", "cum", "scores", "parents", "tokens"):
        setattr(a, f, 64)
    a.groups, a.beams, a.n, a.V, a.eos, a.logits_stride = 2, 4, 8, 1000, -1, 1000
    for k, v in kw.items():
        setattr(a, k, v)
    return cdna4.lib().cdna4_beam_select(ctypes.byref(a), dtype, ws, n, None)


@pytest.mark.parametrize("bad", [
    dict(groups=-1), dict(beams=0), dict(beams=65), dict(beams=-1), dict(V=0), dict(V=-5), dict(V=2 ** 31 - 1), dict(logits_stride=999),
    dict(groups=2 ** 22, beams=4), dict(done=64), dict(done=64, eos=1000), dict(done=64, eos=-1), dict(logits=None), dict(cum=None), dict(scores=None),
    dict(parents=None), dict(tokens=None), dict(logits=65), dict(cum=66), dict(scores=66), dict(parents=66), dict(tokens=66), dict(done=66, eos=1)])
def test_beam_refuses(bad):
    assert beam(**bad) == 1


def test_beam_refuses_sizes_and_workspaces():
    for dt in (cdna4.F64, cdna4.I32, 9, -1):
        assert beam(dtype=dt) == 1
    a = cdna4.BeamArgs(64, 64, None, 64, 64, 64, 2, 4, 0, 1000, -1, 1000)
    assert cdna4.lib().cdna4_beam_select(ctypes.byref(a), cdna4.F16, P, 1 << 40, None) == 1          # n 0
    a.n = 65
    assert cdna4.lib().cdna4_beam_select(ctypes.byref(a), cdna4.F16, P, 1 << 40, None) == 1
    need = cdna4.beam_select_workspace_size(8, 1000, 4, 8)
    assert need > 0 and beam(n=need - 1) == 1 and beam(ws=None) == 1 and beam(ws=ODD8) == 1
    for bad in ((-1, 1000, 4, 8), (8, 0, 4, 8), (8, 1000, 0, 8), (8, 1000, 65, 8), (8, 1000, 4, 0), (8, 1000, 4, 65), (2 ** 24, 1000, 4, 8)):
        assert cdna4.beam_select_workspace_size(*bad) == 0
    assert cdna4.lib().cdna4_beam_select(None, cdna4.F16, P, 1 << 40, None) == 1
    assert beam(groups=0, logits=None, cum=None, scores=None, parents=None, tokens=None, ws=None, n=0) == 0   # nothing to do
    assert beam(dtype=cdna4.F32, logits=66) == 1


@pytest.mark.parametrize("n", [1, 3, 5, 64])
def test_beam_refuses_scores_over_the_cum_of_other_groups(n):
    """scores may be cum where a group has as many of each."""
    a = cdna4.BeamArgs(64, 128, None, 128, 256, 320, 2, 4, n, 1000, -1, 1000)
    assert cdna4.lib().cdna4_beam_select(ctypes.byref(a), cdna4.F16, P, 1 << 40, None) == 1


@pytest.mark.parametrize("bad", [
    dict(groups=-1), dict(beams=0), dict(beams=65), dict(V=0), dict(V=2 ** 31 - 1), dict(logits_stride=999), dict(groups=2 ** 22), dict(done=64, eos=1000),
    dict(done=64, eos=-1), dict(logits=None), dict(cum=None), dict(scores=None), dict(parents=None), dict(tokens=None), dict(logits=65), dict(cum=66),
    dict(scores=66), dict(parents=66), dict(tokens=66), dict(done=66, eos=1), dict(n=0), dict(n=65), dict(dtype=cdna4.F64), dict(ws=None), dict(ws=ODD8),
    dict(n_bytes=600)])
def test_beam_refuses_with_scores_of_their_own(bad):
    """Each by itself, scores and cum apart."""
    a = cdna4.BeamArgs(64, 128, None, 192, 256, 320, 2, 4, 8, 1000, -1, 1000)
    kw = dict(bad)
    dtype, ws, n_bytes = kw.pop("dtype", cdna4.F16), kw.pop("ws", P), kw.pop("n_bytes", 1 << 40)
    for k, v in kw.items():
        setattr(a, k, v)
    assert cdna4.lib().cdna4_beam_select(ctypes.byref(a), dtype, ws, n_bytes, None) == 1


def test_python_refuses_cpu_tensors():
    c = cache()
    x, t = torch.zeros(3, 2, 128, dtype=torch.float16), torch.zeros(3, 4, dtype=torch.int32)
    pool = torch.zeros(cdna4.paged_pool_shape(c), dtype=torch.float16)
    with pytest.raises(ValueError):
        cdna4.rope_append_paged(x, x, x, pool, pool, t, t[:, 0], c)
    with pytest.raises(ValueError):
        cdna4.decode_paged(x, pool, pool, t, t[:, 0], x, c, cdna4.PagedDecodeCfg(2, 3, 1))
    with pytest.raises(ValueError):
        cdna4.paged_reorder(t[:, 0], t, t[:, 0], t[:, 0], t, t[:, 0], pool, pool, c)
    with pytest.raises(ValueError):
        cdna4.beam_select(torch.zeros(4, 10), torch.zeros(4), 4)


def test_token_strides():
    """The C call takes a stride of 0 for packed tokens, so Python passes it only where the stride does not matter."""
    f16, x = torch.float16, torch.zeros(16, 10, 64, dtype=torch.float16)
    stride = lambda t, *shape: cdna4._rows("k", t, f16, -1, shape or tuple(t.shape))
    assert stride(x) == 640 and stride(x[:, 2:5]) == 640 and stride(x[::2, :1]) == 1280 and stride(x[:1]) == 0 and stride(x[:0]) == 0
    assert stride(x[:1, :1].expand(1, 1, 64)) == 0
    for t in (x[:1].expand(16, 10, 64), x[:1, :1].expand(16, 1, 64), x.as_strided((3, 10, 64), (64, 64, 1)), x.as_strided((2, 1, 64), (32, 64, 1)),
              x.as_strided((2, 10, 64), (639, 64, 1))):
        with pytest.raises(ValueError):
            stride(t)
    for t in (x[:, ::2], x[:, :, ::2], x[:, :1].expand(16, 10, 64)):
        with pytest.raises(ValueError):
            stride(t)


def test_tables_rows():
    """Tables whose rows are not as far apart as the kernels read them would name other sequences' pages."""
    take = lambda c, rows, *shape: cdna4._tables("tables", torch.zeros(*shape, dtype=torch.int32), c, rows, -1)
    packed, wide = cache(), cache(table_stride=7)                # max_pages 4
    for ok in ((packed, 3, 3, 4), (packed, 3, 5, 4), (packed, 1, 1, 7), (packed, 3, 12), (packed, 0, 3, 7), (packed, 6, 2, 3, 4), (wide, 3, 3, 7),
               (wide, 1, 1, 4), (wide, 3, 18)):
        take(*ok)
    for bad in ((packed, 3, 3, 7), (packed, 2, 3, 5), (packed, 3, 6, 3), (packed, 1, 5, 2), (packed, 3, 2, 4), (packed, 3, 11), (wide, 3, 3, 8), (wide, 3, 5, 4),
                (wide, 3, 2, 7), (wide, 3, 17)):
        with pytest.raises(ValueError):
            take(*bad)
    with pytest.raises(ValueError):
        cdna4._tables("tables", None, packed, 3, -1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_mxfp4_reference(dtype):
    """Every grid value at every scale is kept; midpoints go to the even code; a block's largest value is off by half a step at most."""
    for e in (-23, -3, 0, 9):
        x = torch.zeros(1, 32, dtype=torch.float64)
        x[0, :8], x[0, 8:16] = GRID * 2.0 ** e, -GRID * 2.0 ** e
        code, scale = quantise(x, dtype)
        assert int(scale) == e + 127 and torch.equal(values(code, scale), x)
    mid = (GRID[1:] + GRID[:-1]) / 2
    x = torch.zeros(1, 32, dtype=torch.float64)
    x[0, :7], x[0, 7] = mid, 6.0
    code, _ = quantise(x, dtype)
    assert code[0, :8].tolist() == [0, 2, 2, 4, 4, 6, 6, 7]
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 64, generator=g).to(dtype)
    code, scale = quantise(x, dtype)
    assert bool(((values(code, scale) - x.double()).abs() <= 2.0 ** (scale.double().repeat_interleave(32, -1) - 127)).all())
    top = x.double().abs().unflatten(-1, (2, 32)).amax(-1)
    assert bool((top < 7 * 2.0 ** (scale.double() - 127)).all()) and bool((top >= 7 * 2.0 ** (scale.double() - 128)).all())
    pool = pack(code.view(4, 16, 64), scale.view(4, 16, 2), 16)
    c, s = unpack(pool, 16, 64)
    assert torch.equal(c.reshape(64, 64), code) and torch.equal(s.reshape(64, 2), scale)


CALLER = r"""
#include <cdna3/attention.hpp>
#include <cdna3/runtime/forward.hpp>
using namespace cdna3;
int main() {
    attn::PagedCache c{128, 2, 64, 10, CDNA4_KV_16, 400, 0};
    attn::PagedDecodeCfg d{8, 3, 1};
    if (attn::decode_paged_workspace_size(c, d) == 0) return 1;
    const __half* h = nullptr;
    const __hip_bfloat16* b = nullptr;
    if (attn::decode_paged(h, h, h, nullptr, nullptr, (__half*)nullptr, c, d, nullptr, 0) != hipErrorInvalidValue) return 2;
    if (attn::decode_paged(b, b, b, nullptr, nullptr, (__hip_bfloat16*)nullptr, c, d, nullptr, 0) != hipErrorInvalidValue) return 3;
    runtime::AppendArgs a{};
    a.T = 1;
    if (runtime::rope_append_paged(a, c, CDNA4_F16) != hipErrorInvalidValue) return 4;
    if (runtime::paged_reorder(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, c, 1, 1) != hipErrorInvalidValue) return 5;
    runtime::BeamArgs s{};
    s.groups = 1;
    if (runtime::beam_select(s, CDNA4_F32, nullptr, 0) != hipErrorInvalidValue) return 6;
    if (runtime::beam_select_workspace_size(4, 1000, 4, 8) == 0) return 7;
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
